// Eviction of the least attended keys from the paged cache.
//
// For every (sequence w, KV head h), of the n = lengths[w] tokens at logical positions
// starts[w] + i, the first `sink` and the last `recent` come first, then the others by
// decreasing mass (NaN after everything else), equal ones by position; the first
// kept = min(n, keep[w]) of that order survive.  Survivors at i < kept stay where they are;
// the i-th hole in front of kept is filled by the i-th survivor behind it.  Attention sums
// over keys in any order and a cached key carries its own rotation, so only these moves are
// needed: every destination is an evicted key and every source lies behind kept, so no move
// reads what another writes.
//
// Two launches: evict_select_kernel (one block per (w, h): the survivors, the moves, the
// moved mass and the map of where each position's token came from), evict_move_kernel
// (copies the K and V rows).
#include "decode.cuh"

#include <cstdio>
#include <cstdlib>

namespace dvb {

struct EvictParams {
    int W, Hkv, BS, maxb, sink, recent;
    int words;  // 32-bit words of a bitmap over a mass row
    int ck, cv; // 16-byte chunks of a K row, of a V row
    int smem_maps;  // the bitmaps lie in shared memory (else in the workspace)
    long long NB, N, cap;
    void* k;
    void* v;
    const float* mass;
    float* mass_out;  // may be `mass`
    int* source;      // may be null
    const int* bt;
    const int* starts;
    const int* lengths;
    const int* keep;
    int* count;       // workspace [W * Hkv] moves of a row
    int2* moves;      // workspace [W * Hkv][N / 2] {to, from}, logical positions
    uint32_t* maps;   // workspace [W * Hkv][2][words] unless smem_maps
};

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;

// Order of a mass as an unsigned integer: larger mass, larger key; -0 equals +0; NaN lowest.
__device__ __forceinline__ uint32_t mass_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix sum of one value per thread over the block, and the total.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* sh, unsigned long long& total) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    unsigned long long incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    __syncthreads();  // sh may still be read from the scan before
    if (lane == 31) sh[wid] = incl;
    __syncthreads();
    unsigned long long before = 0, all = 0;
    for (int i = 0; i < kSelThreads / 32; ++i) {
        const unsigned long long x = sh[i];
        before += i < wid ? x : 0;
        all += x;
    }
    total = all;
    return before + incl - v;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictParams p) {
    extern __shared__ uint32_t dyn[];  // 2 bitmaps, if smem_maps
    __shared__ int hist[kBins];
    __shared__ unsigned long long sh[kSelThreads / 32];
    __shared__ int s_digit, s_above;
    const int tid = threadIdx.x, lane = tid & 31;
    const int row = blockIdx.x, w = row / p.Hkv;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const float* mass = p.mass + (size_t)row * p.N;
    float* mout = p.mass_out + (size_t)row * p.N;
    int* src = p.source ? p.source + (size_t)row * p.N : nullptr;
    const long long start64 = __ldg(p.starts + w), len64 = __ldg(p.lengths + w);
    const long long lim = p.N < p.cap ? p.N : p.cap;  // positions that have a mass and a place in the table
    const int start = start64 < 0 || start64 > lim ? 0 : (int)start64;
    const int n = start64 < 0 || start64 >= lim || len64 <= 0 ? 0 : (int)(len64 < lim - start ? len64 : lim - start);
    const int keep = max(__ldg(p.keep + w), 0), kept = min(n, keep);
    auto key_at = [&](int i) {
        return i < p.sink || i >= n - p.recent ? 0xffffffffu : mass_key(mass[start + i]);
    };
    // ---- the kept-th largest key, 11 + 11 + 10 bits at a time ----
    uint32_t prefix = 0;
    int need = kept;  // survivors still to be found among the keys that share the prefix
    if (kept < n && kept > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kSelThreads) {
                const uint32_t k = key_at(i);
                if (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits))) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1);
            }
            __syncthreads();
            // bins from the top down: thread t holds bins top - 2t, top - 2t - 1
            const int b = kBins - 1 - 2 * tid;
            unsigned long long total;
            const int c0 = hist[b], c1 = hist[b - 1];
            const int above = (int)block_scan((unsigned long long)(c0 + c1), sh, total);
            if (above < need && need <= above + c0) s_digit = b, s_above = above;
            if (above + c0 < need && need <= above + c0 + c1) s_digit = b - 1, s_above = above + c0;
            __syncthreads();
            prefix |= (uint32_t)s_digit << shift;
            need -= s_above;
            __syncthreads();
        }
    }
    // survivors: keys above `prefix`, and the first `need` keys equal to it
    uint32_t* m_keep = p.smem_maps ? dyn : p.maps + (size_t)row * 2 * p.words;
    uint32_t* m_tie = m_keep + p.words;
    const int words = (n + 31) / 32;
    const bool all = kept == n, none = kept == 0;
    for (int i0 = tid - lane; i0 < n; i0 += kSelThreads) {
        const int i = i0 + lane;
        const uint32_t k = i < n && !all && !none ? key_at(i) : 0u;
        const unsigned a = __ballot_sync(0xffffffffu, i < n && !none && (all || k > prefix));
        const unsigned t = __ballot_sync(0xffffffffu, i < n && !all && !none && k == prefix);
        if (lane == 0) m_keep[i0 >> 5] = a, m_tie[i0 >> 5] = t;
    }
    __syncthreads();
    // a thread owns `per` words: first the ties, then holes and movers
    const int per = (words + kSelThreads - 1) / kSelThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);
    unsigned long long total;
    {
        int c = 0;
        for (int x = w0; x < w1; ++x) c += __popc(m_tie[x]);
        int left = need - (int)block_scan((unsigned long long)c, sh, total);
        for (int x = w0; x < w1; ++x) {
            uint32_t t = m_tie[x];
            uint32_t take = 0;
            while (t && left > 0) {
                take |= t & (0u - t);
                t &= t - 1;
                --left;
            }
            m_keep[x] |= take;
        }
    }
    auto below = [&](int x) {  // the bits of word x that lie in front of kept
        const int d = kept - 32 * x;
        return d <= 0 ? 0u : d >= 32 ? 0xffffffffu : (1u << d) - 1;
    };
    int nh = 0, nm = 0;
    for (int x = w0; x < w1; ++x) {
        const uint32_t k = m_keep[x], f = below(x);
        nh += __popc(~k & f);
        nm += __popc(k & ~f);
    }
    const unsigned long long at = block_scan((unsigned long long)nh << 32 | (unsigned)nm, sh, total);
    int ih = (int)(at >> 32), im = (int)(at & 0xffffffffu);
    int2* mv = p.moves + (size_t)row * (p.N / 2);
    for (int x = w0; x < w1; ++x) {
        const uint32_t k = m_keep[x], f = below(x);
        for (uint32_t hole = ~k & f; hole; hole &= hole - 1) mv[ih++].x = start + 32 * x + __ffs(hole) - 1;
        for (uint32_t mover = k & ~f; mover; mover &= mover - 1) mv[im++].y = start + 32 * x + __ffs(mover) - 1;
    }
    const int moved = (int)(total >> 32);
    if (tid == 0) p.count[row] = moved;
    __syncthreads();  // the block's moves and bitmaps are complete
    // ---- mass and source: the moved ones, then the rest ----
    for (int i = tid; i < moved; i += kSelThreads) {
        const int2 m = mv[i];
        mout[m.x] = mass[m.y];
        if (src) src[m.x] = m.y;
    }
    __syncthreads();  // in place: every moved mass is read before the tail is cleared
    const bool in_place = mout == mass;
    for (long long q = tid; q < p.N; q += kSelThreads) {
        const long long i = q - start;
        if (i >= 0 && i < n) {
            if (i >= kept) {
                mout[q] = 0.f;
                if (src) src[q] = -1;
                continue;
            }
            if (!(m_keep[i >> 5] >> (i & 31) & 1u)) continue;  // a filled hole
        }
        if (!in_place) mout[q] = mass[q];
        if (src) src[q] = (int)q;
    }
}

// A warp per move: the lanes copy the 16-byte chunks of the token's K row, then of its V row.
__global__ void __launch_bounds__(256) evict_move_kernel(EvictParams p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row = blockIdx.y, w = row / p.Hkv, h = row - w * p.Hkv, lane = threadIdx.x & 31;
    const int n = __ldcg(p.count + row);
    const int* bt = p.bt + (size_t)w * p.maxb;
    const int2* mv = p.moves + (size_t)row * (p.N / 2);
    for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += gridDim.x * 8) {
        const int2 m = __ldcg(mv + i);
        const int pd = __ldg(bt + m.x / p.BS), ps = __ldg(bt + m.y / p.BS);
        if (pd < 0 || pd >= p.NB || ps < 0 || ps >= p.NB) continue;
        const size_t d = ((size_t)pd * p.BS + m.x % p.BS) * p.Hkv + h, s = ((size_t)ps * p.BS + m.y % p.BS) * p.Hkv + h;
        for (int c = lane; c < p.ck + p.cv; c += 32) {
            if (c < p.ck) static_cast<uint4*>(p.k)[d * p.ck + c] = static_cast<const uint4*>(p.k)[s * p.ck + c];
            else static_cast<uint4*>(p.v)[d * p.cv + c - p.ck] = static_cast<const uint4*>(p.v)[s * p.cv + c - p.ck];
        }
    }
}

// ---------------------------------------------------------------------------------------
// Up to this many bytes of bitmaps a block keeps them in shared memory (rows of 786432
// positions); longer rows have them in the workspace.
constexpr long long kMapSmem = 192 * 1024;

static int evict_validate(const dvattn_evict_args* a) {
    if (!a) return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->dtype < 0 || a->dtype > 2) return DVATTN_ERR_UNSUPPORTED;
    if (a->W < 0 || a->Hkv <= 0 || a->E <= 0 || a->Ev <= 0 || a->block_size <= 0 || a->max_blocks_per_seq < 0 || a->num_blocks < 0 ||
        a->positions < 0 || a->sink < 0 || a->recent < 0)
        return DVATTN_ERR_INVALID_ARGUMENT;
    const int esz = a->dtype == DVATTN_FLOAT32 ? 4 : 2;
    if ((a->E * esz) % 16 || (a->Ev * esz) % 16) return DVATTN_ERR_UNSUPPORTED;
    if (a->positions > 0x7fffffffLL || (long long)a->max_blocks_per_seq * a->block_size > 0x7fffffffLL ||
        (long long)a->W * a->Hkv > 65535)
        return DVATTN_ERR_UNSUPPORTED;
    return DVATTN_OK;
}
static bool evict_nothing(const dvattn_evict_args* a) { return a->W == 0 || a->positions == 0; }

struct EvictLayout {
    size_t count, moves, maps, total;
    int words, smem_maps;
};
static EvictLayout evict_layout(const dvattn_evict_args* a) {
    EvictLayout L;
    const size_t rows = (size_t)a->W * a->Hkv;
    size_t at = 256;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    L.words = (int)((a->positions + 31) / 32);
    L.smem_maps = 8LL * L.words <= kMapSmem;
    L.count = take(4 * rows);
    L.moves = take(8 * rows * (size_t)(a->positions / 2));
    L.maps = take(L.smem_maps ? 0 : 8 * rows * (size_t)L.words);
    L.total = at;
    return L;
}

size_t evict_workspace_size(const dvattn_evict_args* a) {
    if (evict_validate(a) != DVATTN_OK || evict_nothing(a)) return 0;
    return evict_layout(a).total;
}

int evict_launch(const dvattn_evict_args* a, void* workspace, size_t wbytes, cudaStream_t stream) {
    const int st = evict_validate(a);
    if (st != DVATTN_OK) return st;
    if (evict_nothing(a)) return DVATTN_OK;
    if (!a->k_cache || !a->v_cache || !a->mass || !a->mass_out || !a->block_tables || !a->starts || !a->lengths || !a->keep)
        return DVATTN_ERR_INVALID_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(a->k_cache) & 15) || (reinterpret_cast<uintptr_t>(a->v_cache) & 15)) return DVATTN_ERR_INVALID_ARGUMENT;
    const size_t mbytes = 4 * (size_t)a->W * a->Hkv * (size_t)a->positions;
    const uintptr_t mi = reinterpret_cast<uintptr_t>(a->mass), mo = reinterpret_cast<uintptr_t>(a->mass_out);
    if (mi != mo && mi < mo + mbytes && mo < mi + mbytes) return DVATTN_ERR_INVALID_ARGUMENT;  // overlap, not in place
    const EvictLayout L = evict_layout(a);
    if (!workspace || wbytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return DVATTN_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    const int esz = a->dtype == DVATTN_FLOAT32 ? 4 : 2;
    EvictParams p{};
    p.W = a->W; p.Hkv = a->Hkv; p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.NB = a->num_blocks;
    p.sink = a->sink; p.recent = a->recent; p.N = a->positions;
    p.cap = (long long)a->max_blocks_per_seq * a->block_size;
    p.words = L.words; p.smem_maps = L.smem_maps; p.ck = a->E * esz / 16; p.cv = a->Ev * esz / 16;
    p.k = a->k_cache; p.v = a->v_cache; p.mass = a->mass; p.mass_out = a->mass_out; p.source = a->source;
    p.bt = a->block_tables; p.starts = a->starts; p.lengths = a->lengths; p.keep = a->keep;
    p.count = reinterpret_cast<int*>(ws + L.count);
    p.moves = reinterpret_cast<int2*>(ws + L.moves);
    p.maps = reinterpret_cast<uint32_t*>(ws + L.maps);
    const int rows = a->W * a->Hkv;
    const size_t smem = L.smem_maps ? 8 * (size_t)L.words : 0;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaFuncSetAttribute((const void*)&evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMapSmem) != cudaSuccess)
        return DVATTN_ERR_CUDA;
    void* args[] = {&p};
    cudaError_t e = cudaLaunchKernel((const void*)&evict_select_kernel, dim3(rows), dim3(kSelThreads), args, smem, stream);
    if (e == cudaSuccess) {
        // about 8 blocks per SM over all rows, no more than a row's moves can use
        const long long most = (a->positions / 2 + 7) / 8, want = (8LL * sms + rows - 1) / rows;
        const unsigned gx = (unsigned)(want < most ? want : most > 0 ? most : 1);
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cfg.stream = stream;
        cfg.gridDim = dim3(gx, rows);
        cfg.blockDim = dim3(256);
        e = cudaLaunchKernelExC(&cfg, (const void*)&evict_move_kernel, args);
    }
    if (e != cudaSuccess) {
        if (getenv("DVATTN_DEBUG")) fprintf(stderr, "dvattn evict launch: %s\n", cudaGetErrorString(e));
        return DVATTN_ERR_CUDA;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
