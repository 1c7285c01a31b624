// Packed chunked prefill over a paged cache held in 8 bits (q8.cuh).
//
// Calls that the 16-bit attention gives to its tensor-core prefill and whose sequences have many tokens: the pages that
// the call's tokens see are widened to the queries' type in the workspace (value x scale, rounded once: exact in bf16, and in
// f16 within its range, for the scales that the append sets; f16 values past the range saturate), then it runs over them.
// Its products, 4 E flops for every (query head, key) pair, are what bounds it then; widening a key costs
// 2 E (1 + sizeof T) bytes once per KV head, and reading it again.  The same widening inside the
// attention kernel, per window and work item, would be done again for every 16 tokens.  Eight chunks of up to 777 tokens
// behind up to 8192 keys, 32 / 2 heads of 128, bf16: 19 us of 309 (span 3.5, widening 15.5, of which HBM needs 7.5).
//
// All others (32-bit queries, head dims 64 and 256, odd pages, few tokens): the decode attention over the cache as it is
// (decode_q8.cu), its row tiles of 16 or 32 query rows cut from the packed tokens.  1624 tokens of four sequences behind up to 2000
// keys, 32 / 4 heads: 433 us in f32 (head dim 128), 181 in bf16 with head dim 64; 113 tokens of head dim 128 in bf16 56.
//
// Where both can run (kWidenRows): the tiles read a key's byte once for every 16 or 32 query rows of its sequence and KV head, the
// widening five bytes whatever the rows, so the rows of a sequence decide.  The host knows their average.  bf16, head dim 128,
// keys of 2000 positions in front, widened against row tiles: 592 sequences of one token with 64 / 8 heads 3037 us against 578,
// 74 of 8 tokens (64 rows) 399 against 261, 37 of 16 (128 rows) 209 against 250, 10 of 64 137 against 269; 32 / 2 heads, 8 tokens
// (128 rows) 224 against 265, 4 tokens 428 against 284; 8 / 8 heads, 128 tokens 226 against 277, 64 tokens 420 against 276.
// Behind 8000 keys the two meet at 128 rows (721 and 755).  One sequence of many tokens among others of one (64 / 8 heads): 100
// beside 1024 tokens (89 rows on average) 676 against 643, 64 beside 2048 (260 rows) 589 against 1189.
#include "decode.cuh"
#include "q8.cuh"
#include "turns.cuh"

namespace dvb {

namespace {

struct WidenParams {
    int F, W, T, BS, maxb, cap, own_table;  // own_table: page (w, j) of the widened caches is w * maxb + j
    long long NB, chunks;                   // groups of 8 elements of a page of one cache
    int row8;                               // ... of a (token, head) row: 8, 16 or 32
    int Hkv;
    const int* loc;
    const int* L;
    const int* cu;
    const int* bt;
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    int* span;   // [W][F] keys of the turn that a token of the sequence sees
    int* table;  // [W][maxb]
    void* wk;
    void* wv;
};

// A thread per (turn, token): the sequence of token t is the first w with t < cu[w + 1], else 0, as in the
// varlen attention.
__global__ void __launch_bounds__(256) widen_span_kernel(WidenParams p) {
    const int f = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
    int lo = 0, hi = p.W;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (t < __ldg(p.cu + mid + 1)) hi = mid; else lo = mid + 1;
    }
    const int w = lo < p.W ? lo : 0;
    long long off = 0;
    for (int g = 0; g < f; ++g) off += max(__ldg(p.L + g), 0);
    const int v = t < p.T ? turn_seen(__ldg(p.L + f), __ldg(p.loc + (size_t)f * p.T + t), off, p.cap) : 0;
    const unsigned peers = __match_any_sync(0xffffffffu, w);  // a warp's lanes have one sequence or a few
    const int top = __reduce_max_sync(peers, v);
    if (top > 0 && (threadIdx.x & 31) == __ffs(peers) - 1) atomicMax(p.span + (size_t)w * p.F + f, top);
}

template <class T> __device__ __forceinline__ T widened(float x) {
    if constexpr (Elem<T>::dtype == DVATTN_FLOAT16) x = x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x;
    return Elem<T>::from_f(x);
}

// Lane k of a warp looks at page warp + k * warps of the table; then the warp widens those that are seen.
template <class T> __global__ void __launch_bounds__(256) widen_kernel(WidenParams p) {
    const int lane = threadIdx.x & 31;
    const long long warps = (long long)gridDim.x * 8, me = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), all = (long long)p.W * p.maxb;
    for (long long base = 0; base < all; base += 32 * warps) {
        const long long i = base + me + lane * warps;
        int page = -1;
        if (i < all) {
            const int w = (int)(i / p.maxb), j = (int)(i - (long long)w * p.maxb);
            const long long a = (long long)j * p.BS;
            long long off = 0;
            bool seen = false;
            for (int f = 0; f < p.F; ++f) {
                const int n = __ldcg(p.span + (size_t)w * p.F + f);
                seen |= n > 0 && off < a + p.BS && off + n > a;
                off += max(__ldg(p.L + f), 0);
            }
            if (seen) {
                const int g = __ldg(p.bt + i);
                if (g >= 0 && g < p.NB) page = g;
            }
            if (p.own_table) p.table[i] = page >= 0 ? (int)i : -1;
        }
        for (unsigned todo = __ballot_sync(0xffffffffu, page >= 0); todo; todo &= todo - 1) {
            const int src = __ffs(todo) - 1;
            const long long from = __shfl_sync(0xffffffffu, page, src), to = p.own_table ? base + me + src * warps : from;
            // A lane's groups lie 32 apart, whole rows: their heads go round by as many.
            constexpr int U = 4;
            const int step = 32 / p.row8 % p.Hkv;
            int head = lane / p.row8 % p.Hkv;
            const uint2* in[2] = {reinterpret_cast<const uint2*>(p.k) + from * p.chunks, reinterpret_cast<const uint2*>(p.v) + from * p.chunks};
            uint4* out[2] = {static_cast<uint4*>(p.wk) + to * p.chunks * (sizeof(T) / 2), static_cast<uint4*>(p.wv) + to * p.chunks * (sizeof(T) / 2)};
            const float* sc[2] = {p.ks + from * p.Hkv, p.vs + from * p.Hkv};
            for (long long c0 = lane; c0 < p.chunks; c0 += 32 * U) {
                uint2 x[2][U];
                float s[2][U];
#pragma unroll
                for (int u = 0; u < U; ++u, head = head + step < p.Hkv ? head + step : head + step - p.Hkv)
#pragma unroll
                    for (int tensor = 0; tensor < 2; ++tensor)
                        if (c0 + 32 * u < p.chunks) {
                            x[tensor][u] = __ldg(in[tensor] + c0 + 32 * u);
                            s[tensor][u] = __ldg(sc[tensor] + head);
                        }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int tensor = 0; tensor < 2; ++tensor) {
                        const long long c = c0 + 32 * u;
                        if (c >= p.chunks) continue;
                        alignas(16) T y[8];
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const uint32_t word = b < 2 ? x[tensor][u].x : x[tensor][u].y;
                            const uint32_t f = b & 1 ? e4m3x2_hi_to_f16x2(word) : e4m3x2_to_f16x2(word);
                            const __half2 h = *reinterpret_cast<const __half2*>(&f);
                            y[2 * b] = widened<T>(__low2float(h) * s[tensor][u]);
                            y[2 * b + 1] = widened<T>(__high2float(h) * s[tensor][u]);
                        }
#pragma unroll
                        for (int b = 0; b < (int)sizeof(T) / 2; ++b) out[tensor][c * (sizeof(T) / 2) + b] = reinterpret_cast<const uint4*>(y)[b];
                    }
            }
        }
    }
}

constexpr int kWidenRows = 128;  // query rows of a sequence and KV head, on average, from which pages are widened (file comment)

// Bytes of widened pages that a call asks for at most: the pages of the pool, or of the batch's tables, take up to twice the pool's bytes,
// seen or not, which a GPU that a large pool fills does not have.  Calls that would need more run on the row tiles, in 256 MB.
constexpr size_t kMostWidened = 16ull << 30;

size_t up(size_t x) { return (x + 255) / 256 * 256; }

struct WidenLayout {
    size_t own, span, table, wk, wv, total;
    long long pages;
    bool own_table;
    dvattn_varlen_args wide;  // the call over the widened caches
};
// false: not a call for the tensor-core prefill
bool widen_layout(const dvattn_varlen_args* a, WidenLayout& L) {
    if (!prefill_forced() && (long long)a->T * (a->Hq / a->Hkv) < (long long)kWidenRows * a->W) return false;
    const long long mine = (long long)a->W * a->max_blocks_per_seq;
    L.own_table = mine < a->num_blocks;
    L.pages = L.own_table ? mine : a->num_blocks;
    L.wide = *a;
    L.wide.num_blocks = L.pages;
    if (!prefill_eligible(&L.wide)) return false;
    if ((long long)a->max_blocks_per_seq * a->block_size > kMostPositions) return false;  // windows there pass 32 bits in the prefill
    L.own = prefill_workspace_size(&L.wide);
    const size_t cache = (size_t)L.pages * a->block_size * a->Hkv * a->E * 2;
    if (2 * cache > kMostWidened) return false;
    L.span = up(L.own);
    L.table = L.span + up(4 * (size_t)a->W * a->F);
    L.wk = L.table + (L.own_table ? up(4 * (size_t)mine) : 0);
    L.wv = L.wk + up(cache);
    L.total = L.wv + up(cache);
    return true;
}
// A call of one token for each sequence.
dvattn_paged_args tokens_of(const dvattn_varlen_args* a) {
    dvattn_paged_args v{};
    v.dtype = a->dtype; v.F = a->F; v.W = a->T; v.Hq = a->Hq; v.Hkv = a->Hkv; v.E = a->E; v.Ev = a->Ev; v.S = 1; v.R = a->R;
    v.block_size = a->block_size; v.max_blocks_per_seq = a->max_blocks_per_seq; v.num_blocks = a->num_blocks; v.scale = a->scale;
    v.out = a->out; v.queries = a->queries; v.cosines = a->cosines; v.sines = a->sines; v.locations = a->locations;
    v.fragment_lengths = a->fragment_lengths; v.k_cache = a->k_cache; v.v_cache = a->v_cache; v.block_tables = a->block_tables;
    v.lse_out = a->lse_out; v.out_f32 = a->out_f32;
    return v;
}
int widen_validate(const dvattn_varlen_args* a) {
    if (!a || a->W < 0 || a->T < 0 || a->num_blocks < 0) return DVATTN_ERR_INVALID_ARGUMENT;
    const dvattn_paged_args v = tokens_of(a);
    const int st = decode_validate(&v);
    if (st != DVATTN_OK) return st;
    // tables are indexed in 32 bits where they are the workspace's; turns are a grid's y; row tiles, and one more for every
    // sequence, are counted in 32 bits
    return (long long)a->W * a->max_blocks_per_seq > 0x7fffffffLL || a->F > 65535 ||
                   (long long)a->T * (a->Hq / a->Hkv) > 0x7fffff00LL || a->W > 1 << 30
               ? DVATTN_ERR_UNSUPPORTED : DVATTN_OK;
}

}  // namespace

size_t varlen_q8_workspace_size(const dvattn_varlen_args* a) {
    if (widen_validate(a) != DVATTN_OK || a->T == 0 || a->Hq == 0) return 0;
    WidenLayout L;
    if (widen_layout(a, L)) return L.total;
    const dvattn_paged_args v = tokens_of(a);
    return packed_q8_workspace_size(&v, a->cu_seqlens_q, a->W);
}

int varlen_q8_launch(const dvattn_varlen_args* a, const dvattn_q8_scales* sc, void* workspace, size_t wbytes, cudaStream_t stream) {
    int st = widen_validate(a);
    if (st != DVATTN_OK) return st;
    if (!sc) return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->T == 0 || a->Hq == 0) return DVATTN_OK;
    const bool cached = a->W > 0 && a->max_blocks_per_seq > 0 && a->num_blocks > 0;
    if (!a->out || !a->queries || !a->cu_seqlens_q || !a->k_cache || !a->v_cache || !a->block_tables ||
        (a->F > 0 && (!a->locations || !a->fragment_lengths)) || (a->R > 0 && (!a->cosines || !a->sines)) ||
        (cached && (!sc->k_scales || !sc->v_scales)))
        return DVATTN_ERR_INVALID_ARGUMENT;
    for (const void* x : {a->queries, a->k_cache, a->v_cache, (const void*)a->out, (const void*)a->out_f32})
        if (reinterpret_cast<uintptr_t>(x) & 15) return DVATTN_ERR_INVALID_ARGUMENT;
    WidenLayout L;
    if (!widen_layout(a, L)) {
        const dvattn_paged_args v = tokens_of(a);
        return packed_q8_launch(&v, a->cu_seqlens_q, a->W, sc, workspace, wbytes, stream);
    }
    if (!workspace || wbytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return DVATTN_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    L.wide.k_cache = ws + L.wk;
    L.wide.v_cache = ws + L.wv;
    if (L.own_table) L.wide.block_tables = reinterpret_cast<int*>(ws + L.table);
    if (cached && a->F > 0) {
        WidenParams p{};
        p.F = a->F; p.W = a->W; p.T = a->T; p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.NB = a->num_blocks; p.Hkv = a->Hkv;
        const long long cap = (long long)a->max_blocks_per_seq * a->block_size;
        p.cap = cap > 0x7fffffffLL ? 0x7fffffff : (int)cap;
        p.own_table = L.own_table;
        p.row8 = a->E / 8;
        p.chunks = (long long)a->block_size * a->Hkv * p.row8;
        p.loc = a->locations; p.L = a->fragment_lengths; p.cu = a->cu_seqlens_q; p.bt = a->block_tables;
        p.k = static_cast<const uint8_t*>(a->k_cache); p.v = static_cast<const uint8_t*>(a->v_cache);
        p.ks = sc->k_scales; p.vs = sc->v_scales;
        p.span = reinterpret_cast<int*>(ws + L.span);
        p.table = reinterpret_cast<int*>(ws + L.table);
        p.wk = ws + L.wk; p.wv = ws + L.wv;
        int dev = 0, sms = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
            cudaMemsetAsync(p.span, 0, 4 * (size_t)a->W * a->F, stream) != cudaSuccess)
            return DVATTN_ERR_CUDA;
        widen_span_kernel<<<dim3((unsigned)((a->T + 255) / 256), (unsigned)a->F), 256, 0, stream>>>(p);
        const long long want = ((long long)a->W * a->max_blocks_per_seq + 7) / 8;
        const unsigned grid = (unsigned)(want < 4LL * sms ? want : 4LL * sms);
        if (a->dtype == DVATTN_FLOAT16) widen_kernel<__half><<<grid, 256, 0, stream>>>(p);
        else widen_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(p);
        if (cudaGetLastError() != cudaSuccess) return DVATTN_ERR_CUDA;
    }
    return varlen_launch(&L.wide, workspace, L.own, stream, DVATTN_PHASE_ALL);
}

}  // namespace dvb
