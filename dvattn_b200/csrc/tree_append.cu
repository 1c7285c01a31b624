// Append of a drafted tree's accepted tokens to the paged cache (the step after a verification).
//
// Entry i < counts[w] of worker w takes token t = accepted[w][i] of the tree and goes to logical
// position positions[w] + i: its V rows as they are, its K rows rotated as apply_rotary_pos_emb
// does it, by the bits of the paged append (append.cu): with full-width cos/sin rows c, s and
// h = R / 2, o[e] = x[e] c[e] - x[e + h] s[e], o[e + h] = x[e + h] c[e + h] + x[e] s[e + h] for
// e < h, o[e] = x[e] for e >= R; products and sum rounded separately, one rounding to T.
// An entry whose token, position or page does not exist is skipped.
//
// A warp per (entry, part): rotated pairs of 16-byte chunks (e, e + h), one a lane, or copied
// chunks, kCopies a lane, all loads in flight together.  The first reads of a warp's chain
// (count, token, position) are one round trip, the next (page, rows, cos, sin) another.
//
// Bound: few tokens, the launch and these two (32 sequences of up to 4 accepted tokens: 6 us);
// many, HBM: 44 MB, up to 37 of 64 tokens for each of 256 sequences, take 18.4 us, 37% of its copy
// rate (23 with a warp per entry; two copied chunks a lane, a pair of pairs, half as many blocks
// per SM, or a warp that reads its next entry ahead are no faster).
#include "decode.cuh"

namespace dvb {

struct TreeAppendParams {
    int W, Hkv, E, Ev, n, m, R, BS, maxb;  // n tokens of a tree, m entries of a worker
    int pairs;                             // rotated pairs of chunks of a K row (0: the K rows go element by element)
    int copies;                            // copied chunks of a head's K and V rows
    int parts_k, parts;                    // parts of an entry that rotate, all
    long long NB;
    void* k_cache;
    void* v_cache;
    const void* keys;
    const void* values;
    const float* cos;
    const float* sin;
    const int* bt;
    const int* pos;
    const int* cnt;
    const int* acc;
};

constexpr int kCopies = 4;
constexpr int kThreads = 128, kWarps = kThreads / 32, kBlocks = 8;  // blocks of an SM

template <class T> __global__ void __launch_bounds__(kThreads, kBlocks) tree_append_kernel(TreeAppendParams p) {
    constexpr int PER = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, h = p.R >> 1;
    const int ck = p.E / PER, cv = p.Ev / PER;
    const long long tasks = (long long)p.W * p.m * p.parts;
    for (long long task = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); task < tasks; task += (long long)gridDim.x * kWarps) {
        const int wi = (int)(task / p.parts), part = (int)(task - (long long)wi * p.parts);
        const int w = wi / p.m, i = wi - w * p.m;
        const int cnt = p.cnt ? __ldg(p.cnt + w) : p.m, t = __ldg(p.acc + wi);
        const long long at = (long long)__ldg(p.pos + w) + i;
        if (i >= cnt || t < 0 || t >= p.n || at < 0 || at >= (long long)p.maxb * p.BS) continue;
        const int page = __ldg(p.bt + (size_t)w * p.maxb + (int)at / p.BS);
        const bool there = page >= 0 && page < p.NB;
        const size_t slot = ((size_t)page * p.BS + (int)at % p.BS) * p.Hkv;
        const size_t row0 = (size_t)w * p.Hkv * p.n + t;  // of head 0; head hh: + hh n
        const float* cr = p.cos + ((size_t)w * p.n + t) * p.R;
        const float* sr = p.sin + ((size_t)w * p.n + t) * p.R;
        const T* keys = static_cast<const T*>(p.keys);
        T* kc = static_cast<T*>(p.k_cache);
        if (part >= p.parts_k) {  // ---- copies: of each head the K chunks past R, then the V chunks ----
            const int units = p.Hkv * p.copies, kcopies = p.copies - cv;
            uint4 v[kCopies];
            uint4* dst[kCopies] = {};
#pragma unroll
            for (int u = 0; u < kCopies; ++u) {
                const int j = (part - p.parts_k) * 32 * kCopies + 32 * u + lane;
                if (j >= units) break;
                const int hh = j / p.copies, c = j - hh * p.copies - kcopies;
                const size_t row = row0 + (size_t)hh * p.n;
                const bool k = c < 0;
                const int e = k ? (ck + c) * PER : c * PER;
                v[u] = __ldg(reinterpret_cast<const uint4*>(k ? keys + row * p.E + e : static_cast<const T*>(p.values) + row * p.Ev + e));
                dst[u] = reinterpret_cast<uint4*>(k ? kc + (slot + hh) * p.E + e : static_cast<T*>(p.v_cache) + (slot + hh) * p.Ev + e);
            }
            if (there)
#pragma unroll
                for (int u = 0; u < kCopies; ++u)
                    if (dst[u]) *dst[u] = v[u];
        } else if (p.pairs) {  // ---- rotated pairs of chunks ----
            const int j = part * 32 + lane, hh = j / p.pairs, e = (j - hh * p.pairs) * PER;
            if (hh < p.Hkv) {
                const T* x = keys + (row0 + (size_t)hh * p.n) * p.E + e;
                uint4 lo = __ldg(reinterpret_cast<const uint4*>(x)), hi = __ldg(reinterpret_cast<const uint4*>(x + h));
                float c0[PER], s0[PER], c1[PER], s1[PER];
#pragma unroll
                for (int y = 0; y < PER; y += 4) {
                    *reinterpret_cast<float4*>(c0 + y) = __ldg(reinterpret_cast<const float4*>(cr + e + y));
                    *reinterpret_cast<float4*>(s0 + y) = __ldg(reinterpret_cast<const float4*>(sr + e + y));
                    *reinterpret_cast<float4*>(c1 + y) = __ldg(reinterpret_cast<const float4*>(cr + e + h + y));
                    *reinterpret_cast<float4*>(s1 + y) = __ldg(reinterpret_cast<const float4*>(sr + e + h + y));
                }
                T* a = reinterpret_cast<T*>(&lo);
                T* b = reinterpret_cast<T*>(&hi);
#pragma unroll
                for (int y = 0; y < PER; ++y) {
                    const float va = Elem<T>::to_f(a[y]), vb = Elem<T>::to_f(b[y]);
                    a[y] = Elem<T>::from_f(__fadd_rn(__fmul_rn(va, c0[y]), __fmul_rn(-vb, s0[y])));
                    b[y] = Elem<T>::from_f(__fadd_rn(__fmul_rn(vb, c1[y]), __fmul_rn(va, s1[y])));
                }
                if (there) {
                    T* dst = kc + (slot + hh) * p.E + e;
                    *reinterpret_cast<uint4*>(dst) = lo;
                    *reinterpret_cast<uint4*>(dst + h) = hi;
                }
            }
        } else if (there) {  // ---- K chunks element by element: halves that are not whole chunks, unaligned cos or sin ----
            const int j = part * 32 + lane, hh = j / ck, e0 = (j - hh * ck) * PER;
            if (hh < p.Hkv) {
                const T* x = keys + (row0 + (size_t)hh * p.n) * p.E;
                alignas(16) T o[PER];
#pragma unroll
                for (int y = 0; y < PER; ++y) {
                    const int e = e0 + y;
                    const float v = Elem<T>::to_f(x[e]);
                    o[y] = x[e];
                    if (e < p.R) {
                        const float z = e < h ? -Elem<T>::to_f(x[e + h]) : Elem<T>::to_f(x[e - h]);
                        o[y] = Elem<T>::from_f(__fadd_rn(__fmul_rn(v, __ldg(cr + e)), __fmul_rn(z, __ldg(sr + e))));
                    }
                }
                *reinterpret_cast<uint4*>(kc + (slot + hh) * p.E + e0) = *reinterpret_cast<const uint4*>(o);
            }
        }
    }
}

int tree_append_launch(const dvattn_tree_append_args* a, cudaStream_t stream) {
    if (!a || a->A < 0) return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->dtype < 0 || a->dtype > 2) return DVATTN_ERR_UNSUPPORTED;
    if (a->W < 0 || a->S < 0 || a->Hkv <= 0 || a->E <= 0 || a->Ev <= 0 || a->R < 0 || a->R > a->E || (a->R & 1) || a->block_size <= 0 ||
        a->max_blocks_per_seq < 0 || a->num_blocks < 0)
        return DVATTN_ERR_INVALID_ARGUMENT;
    const int esz = a->dtype == DVATTN_FLOAT32 ? 4 : 2, per = 16 / esz;
    if (a->E % per || a->Ev % per) return DVATTN_ERR_UNSUPPORTED;
    if (a->W == 0 || a->S == 0 || a->A == 0) return DVATTN_OK;
    if ((long long)a->W * a->S >= (1LL << 31) || (long long)a->W * a->A >= (1LL << 31) ||
        (long long)a->max_blocks_per_seq * a->block_size >= (1LL << 31))
        return DVATTN_ERR_UNSUPPORTED;
    if (!a->k_cache || !a->v_cache || !a->draft_keys || !a->draft_values || !a->block_tables || !a->positions || !a->accepted ||
        (a->R > 0 && (!a->cosines || !a->sines)))
        return DVATTN_ERR_INVALID_ARGUMENT;
    for (const void* q : {(const void*)a->k_cache, (const void*)a->v_cache, a->draft_keys, a->draft_values})
        if (reinterpret_cast<uintptr_t>(q) & 15) return DVATTN_ERR_INVALID_ARGUMENT;
    TreeAppendParams p{};
    p.W = a->W; p.Hkv = a->Hkv; p.E = a->E; p.Ev = a->Ev; p.n = a->S; p.m = a->A; p.R = a->R;
    p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.NB = a->num_blocks;
    p.k_cache = a->k_cache; p.v_cache = a->v_cache; p.keys = a->draft_keys; p.values = a->draft_values;
    p.cos = a->cosines; p.sin = a->sines; p.bt = a->block_tables; p.pos = a->positions; p.cnt = a->counts; p.acc = a->accepted;
    const bool whole = a->R / 2 % per == 0 && !((reinterpret_cast<uintptr_t>(a->cosines) | reinterpret_cast<uintptr_t>(a->sines)) & 15);
    p.pairs = whole ? a->R / 2 / per : 0;
    // R = 0: every K chunk is a copy
    const int ck = a->E / per, rotated = a->R == 0 ? 0 : whole ? 2 * p.pairs : ck;
    p.copies = ck - rotated + a->Ev / per;
    const long long units_k = (long long)a->Hkv * (p.pairs ? p.pairs : rotated), units_c = (long long)a->Hkv * p.copies;
    if (units_c >= (1LL << 30) || units_k >= (1LL << 30)) return DVATTN_ERR_UNSUPPORTED;
    p.parts_k = (int)((units_k + 31) / 32);
    p.parts = p.parts_k + (int)((units_c + 32 * kCopies - 1) / (32 * kCopies));
    const long long blocks = ((long long)a->W * a->A * p.parts + kWarps - 1) / kWarps;
    const int grid = (int)(blocks < (1LL << 30) ? blocks : 1LL << 30);
    switch (a->dtype) {
        case DVATTN_FLOAT16: tree_append_kernel<__half><<<grid, kThreads, 0, stream>>>(p); break;
        case DVATTN_BFLOAT16: tree_append_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p); break;
        default: tree_append_kernel<float><<<grid, kThreads, 0, stream>>>(p); break;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
