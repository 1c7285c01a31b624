// Attention of a tree of drafted tokens over the paged multi-turn cache, verified in one
// pass (tree.cuh: the items; turns.cuh: the work split).
//
//   out[w, h, s] = sum_j softmax_j(scale * q . k_j) v_j  over the cached keys that
//   (w, s) sees in every turn (q rotated for that turn) and the drafted keys of s's
//   ancestors and of s itself (q and key rotated with their own angles in the last turn, the key
//   as tree_append.cu writes it).
//
// Three launches: tree_prep_kernel (ancestor sets, visible spans, rotated drafted keys),
// the attention kernel, and tree_merge_kernel, each a programmatic dependent of the one
// before it.  The running maximum and sum, the scores and the output accumulate in 32 bits.
#include "tree.cuh"

#include <cstdio>
#include <cstdlib>

namespace dvb {

// ---- prep ---------------------------------------------------------------------------
// Block (w, 0) finds sequence w's ancestor sets, what each token sees of each turn and the
// spans; the others rotate its queries for every turn and its drafted keys, once for all the
// CTAs that read them, and copy its drafted values without infinities and NaN (tree_tc.cu).  Reads
// and writes (F + 1 parts of Hkv rows) a few percent of a call's bytes, 6 us for one turn and one
// more per turn; done by the attention kernel's own threads, the rotation stood between two pieces
// of its work for 5 us and more.
constexpr int kPrepChunks = 256;  // 16-byte chunks of a rotating block

template <class T>
__global__ void __launch_bounds__(256, 4) tree_prep_kernel(TreeParams p, int E) {
    extern __shared__ int par[];  // [S] parents, then [S] whether a token is there
    asm volatile("griddepcontrol.wait;" ::: "memory");  // a programmatic dependent of whatever is before it
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int w = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    if (blockIdx.y == 0) {
        __shared__ int part[8];
        int* there = par + p.S;
        if (w == 0 && tid < 4) p.header[tid] = 0;
        for (int j = tid; j < p.Hkv; j += 256) p.odd_any[w * p.Hkv + j] = 0;
        for (int j = tid; j < p.S; j += 256) par[j] = __ldg(p.parents + (size_t)w * p.S + j);
        __syncthreads();
        // a token is there if its line of parents, each before its child, ends at -1
        for (int j = tid; j < p.S; j += 256) {
            int c = j;
            while (c >= 0 && par[c] < c && par[c] >= -1) c = par[c];
            there[j] = c == -1;
            uint32_t* a = p.anc + ((size_t)w * p.S + j) * p.SW;
            c = c == -1 ? j : -1;
            for (int word = p.SW - 1; word >= 0; --word) {
                uint32_t bits = 0;
                while (c >= 32 * word) {  // c < 32 * (word + 1) here: parents come before
                    bits |= 1u << (c & 31);
                    c = par[c];
                    if (c < 0) break;
                }
                a[word] = bits;
            }
        }
        __syncthreads();
        // a warp per turn
        long long off = 0;
        int nw = 0, at = 0;  // `off`: the first position of turn `at`
        for (int f = wid; f < p.F; f += 8) {
            for (; at < f; ++at) off += max(__ldg(p.L + at), 0);
            const int Lf = __ldg(p.L + f);
            int v = 0, least = 0x7fffffff;
            for (int s = lane; s < p.S; s += 32) {
                const size_t x = ((size_t)f * p.W + w) * p.S + s;
                const int n = there[s] ? turn_seen(Lf, __ldg(p.loc + x), off, p.cap) : 0;
                p.lim[x] = n;
                v = max(v, n);
                if (there[s]) least = min(least, n);
            }
            v = __reduce_max_sync(0xffffffffu, v);
            least = __reduce_min_sync(0xffffffffu, least);
            const int first = v > 0 ? (int)off : 0;  // below cap where a key is seen
            if (lane == 0) {
                p.span[(size_t)w * p.F + f] = make_int2(v, least < v ? first | (int)0x80000000 : first);
                p.same[(size_t)w * p.F + f] = least;
            }
            nw += turn_windows(p, v, first);
        }
        if (lane == 0) part[wid] = nw;
        __syncthreads();
        if (tid == 0) {
            for (int x = 1; x < 8; ++x) nw += part[x];
            p.nwin[w] = nw + (p.S + p.kt - 1) / p.kt;
        }
        return;
    }
    // a chunk a thread: of the drafted keys [Hkv][S], for the last turn, of the queries [Hkv][rows], for
    // every turn, or of the drafted values
    const int keys = p.Hkv * p.S, per = E * (int)sizeof(T) / 16, all = (keys + p.Hkv * p.rows) * per;
    int c = (blockIdx.y - 1) * kPrepChunks + tid;
    const int copies = (all + kPrepChunks - 1) / kPrepChunks;  // the first block with values
    if (sizeof(T) == 2 && (int)blockIdx.y > copies) {
        c -= copies * kPrepChunks;
        if (c >= keys * per) return;
        const size_t at = (size_t)w * keys * per + c;
        uint4 v = __ldg(static_cast<const uint4*>(p.dv) + at);
        if constexpr (sizeof(T) == 2) {  // a row's `per` lanes (8, 16 or 32) are neighbours
            const unsigned group = per == 32 ? 0xffffffffu : ((1u << per) - 1) << (lane & ~(per - 1));
            const unsigned any = __ballot_sync(group, make_finite<T>(v));
            static_cast<uint4*>(p.dvr)[at] = v;
            if (lane % per == 0) p.odd[at / per] = any != 0;
        }
        return;
    }
    if (c >= all) return;
    const int x = c / per, e0 = (c - x * per) * RotateChunk<T>::PER;
    const bool key = x < keys;
    const int y = x - keys, h = y / p.rows, r = y - h * p.rows, s = key ? x % p.S : r / p.G;
    const T* src = key ? static_cast<const T*>(p.dk) + ((size_t)w * keys + x) * E
                       : static_cast<const T*>(p.q) + (((size_t)w * p.Hq + h * p.G + r - s * p.G) * p.S + s) * E;
    T* dst = key ? static_cast<T*>(p.dkr) + ((size_t)w * keys + x) * E : static_cast<T*>(p.qr) + (((size_t)w * p.Hkv + h) * p.rows + r) * E;
    RotateChunk<T> ch;
    ch.load_row(src, e0, p.R, p.rot_vec, key);
    int f = key ? p.F - 1 : 0;
    for (size_t angle = (((size_t)f * p.W + w) * p.S + s) * p.R; f < p.F; ++f) {
        ch.load_angles(dst, p.cos + angle, p.sin + angle, p.R, p.rot_vec);
        ch.store(p.R, p.rot_vec);
        dst += (size_t)p.W * p.Hkv * p.rows * E;
        angle += (size_t)p.W * p.S * p.R;
    }
}

// ---- CUDA-core attention, 32-bit types -----------------------------------------------------
// 32 rows x 32 keys per step, 8 warps of 4 rows.  Scores: a lane per key, q rows broadcast
// from shared memory; output: a lane per E / 32 columns.  K and V tiles are double-buffered
// with cp.async (zero-filled where a key is not seen, so what lies there never matters).
template <int E> struct SimtCfg {
    static constexpr int KT = 32, MI = 32, THREADS = 256;
    static constexpr int ROW = E * 4 + 16;  // padded row, bytes
    static constexpr size_t SMEM = (size_t)MI * (E + 4) * 4 + 4 * (size_t)KT * ROW + (size_t)MI * (KT + 4) * 4;
};

// key (f, l) of KV head h: its address, or null where there is none to read
__device__ __forceinline__ const float* tree_row(const TreeParams& p, const void* cache, const void* draft, int E, int w, int h,
                                                 const SplitWin& win, int l) {
    if (win.f == p.F) {
        // a drafted token that is not there is read as zeros
        if (!(__ldcg(p.anc + ((size_t)w * p.S + l) * p.SW + (l >> 5)) >> (l & 31) & 1u)) return nullptr;
        return static_cast<const float*>(draft) + (((size_t)w * p.Hkv + h) * p.S + l) * E;
    }
    const int pos = win.off + l;
    const int page = __ldg(p.bt + (size_t)w * p.maxb + pos / p.BS);
    if (page < 0 || page >= p.NB) return nullptr;
    return static_cast<const float*>(cache) + (((size_t)page * p.BS + pos % p.BS) * p.Hkv + h) * E;
}

template <int N> __device__ __forceinline__ void load_n(const float* src, float (&v)[N]) {  // N * 4 bytes aligned, up to 16
    if constexpr (N == 2) {
        const float2 x = *reinterpret_cast<const float2*>(src);
        v[0] = x.x, v[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(src + i);
            v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
        }
    }
}

template <int E> __global__ void __launch_bounds__(SimtCfg<E>::THREADS) tree_simt_kernel(TreeParams p) {
    using C = SimtCfg<E>;
    constexpr int KT = C::KT, MI = C::MI, ROW = C::ROW, CH = E / 4, VC = E / 32;
    extern __shared__ __align__(16) uint8_t smem[];
    float* sQ = reinterpret_cast<float*>(smem);                        // [MI][E + 4]
    uint8_t* sK = smem + (size_t)MI * (E + 4) * 4;                     // [2][KT] rows
    uint8_t* sV = sK + 2 * KT * ROW;                                   // [2][KT] rows
    float* sP = reinterpret_cast<float*>(sV + 2 * KT * ROW);           // [MI][KT + 4]
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // see tree_tc_kernel
    const int g = blockIdx.x / p.Hkv, h = blockIdx.x - g * p.Hkv;
    SplitWalk walk;
    walk.place(p, lane, g);
    const int rows = p.rows;
    SplitPiece pc;
    while (walk.next(p, pc)) {
        SplitWin ld, win;
        ld.start(p, pc.w);
        win.start(p, pc.w);
        auto load = [&](int i, int st) {
            ld.seek(p, pc.w, i);
            for (int c = tid; c < KT * CH; c += C::THREADS) {
                const int r = c / CH, ch = c - r * CH;
                const float* kp = nullptr;
                const float* vp = nullptr;
                if (r < ld.n) {
                    kp = tree_row(p, p.k, p.dkr, E, pc.w, h, ld, ld.k0 + r);
                    vp = tree_row(p, p.v, p.dv, E, pc.w, h, ld, ld.k0 + r);
                }
                cp_async16_zfill(smem_u32(sK + (st * KT + r) * ROW + ch * 16), kp ? kp + ch * 4 : static_cast<const float*>(p.k), kp ? 16 : 0);
                cp_async16_zfill(smem_u32(sV + (st * KT + r) * ROW + ch * 16), vp ? vp + ch * 4 : static_cast<const float*>(p.v), vp ? 16 : 0);
            }
            cp_async_commit();
        };
        float m[4], l[4], o[4][VC];
        int lim[4], tok[4];  // the rows' tokens and the keys they see in the window's turn
        uint32_t there = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = neg_inf();
            l[i] = 0.f;
            const int r = pc.t * MI + wid * 4 + i;
            tok[i] = r < rows ? r / p.G : -1;
            if (tok[i] >= 0 && (__ldcg(p.anc + ((size_t)pc.w * p.S + tok[i]) * p.SW + (tok[i] >> 5)) >> (tok[i] & 31) & 1u)) there |= 1u << i;
#pragma unroll
            for (int c = 0; c < VC; ++c) o[i][c] = 0.f;
        }
        int turn = -1;
        load(pc.i0, 0);
        for (int i = pc.i0; i < pc.i1; ++i) {
            const int st = (i - pc.i0) & 1;
            if (i + 1 < pc.i1) {
                load(i + 1, st ^ 1);
                cp_async_wait<1>();
            } else {
                cp_async_wait<0>();
            }
            win.seek(p, pc.w, i);
            const int qt = win.f < p.F ? win.f : p.F - 1;  // the turn whose rotation q takes
            if (qt != turn) {
                turn = qt;
                const float* qr = static_cast<const float*>(p.qr) + (((size_t)qt * p.W + pc.w) * p.Hkv + h) * p.rows * E;
                for (int c = tid; c < MI * E; c += C::THREADS) {
                    const int r = c / E, e = c - r * E, rr = pc.t * MI + r;
                    sQ[r * (E + 4) + e] = rr < p.rows ? __ldcg(qr + (size_t)rr * E + e) : 0.f;
                }
            }
            if (win.f < p.F)
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    lim[a] = there >> a & 1u ? __ldcg(p.lim + ((size_t)win.f * p.W + pc.w) * p.S + tok[a]) : 0;
            __syncthreads();
            // scores of this warp's 4 rows and the lane's key
            float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int ch = 0; ch < CH; ++ch) {
                float kv[4];
                load_n(reinterpret_cast<const float*>(sK + (st * KT + lane) * ROW + ch * 16), kv);
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const float4 q4 = *reinterpret_cast<const float4*>(sQ + (wid * 4 + a) * (E + 4) + ch * 4);
                    sc[a] = fmaf(q4.x, kv[0], sc[a]);
                    sc[a] = fmaf(q4.y, kv[1], sc[a]);
                    sc[a] = fmaf(q4.z, kv[2], sc[a]);
                    sc[a] = fmaf(q4.w, kv[3], sc[a]);
                }
            }
            const int key = win.k0 + lane;
            uint32_t seen[4];  // the window's keys that a row sees
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                bool sees = false;
                if (lane < win.n && (there >> a & 1u))
                    sees = win.f < p.F ? key < lim[a]
                                       : (__ldcg(p.anc + ((size_t)pc.w * p.S + tok[a]) * p.SW + (key >> 5)) >> (key & 31) & 1u) != 0;
                seen[a] = __ballot_sync(0xffffffffu, sees);
                const float x = sees ? sc[a] * p.scale_log2 : neg_inf();
                float mx = x;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                mx = fmaxf(mx, m[a]);
                const float mu = mx == neg_inf() ? 0.f : mx;
                const float e = fast_exp2(x - mu), alpha = fast_exp2(m[a] - mu);
                float sum = e;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                l[a] = l[a] * alpha + sum;
                m[a] = mx;
                sP[(wid * 4 + a) * (KT + 4) + lane] = e;
#pragma unroll
                for (int c = 0; c < VC; ++c) o[a][c] *= alpha;
            }
            __syncwarp();
#pragma unroll 2
            for (int k4 = 0; k4 < KT; k4 += 4) {
                float pr[4][4];
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    *reinterpret_cast<float4*>(pr[a]) = *reinterpret_cast<const float4*>(sP + (wid * 4 + a) * (KT + 4) + k4);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    float vv[VC];
                    load_n(reinterpret_cast<const float*>(sV + (st * KT + k4 + u) * ROW) + lane * VC, vv);
                    // a row that does not see the key takes nothing of it: 0 * NaN is NaN
#pragma unroll
                    for (int a = 0; a < 4; ++a)
                        if (seen[a] >> (k4 + u) & 1u)
#pragma unroll
                            for (int c = 0; c < VC; ++c) o[a][c] = fmaf(pr[a][u], vv[c], o[a][c]);
                }
            }
            __syncthreads();
        }
        // the piece's result
        const bool whole = pc.whole();
        const size_t slot = (size_t)blockIdx.x * 2 + pc.slot();
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            if (tok[a] < 0) continue;
            const float inv = l[a] > 0.f ? 1.f / l[a] : l[a] == 0.f ? 0.f : l[a];
            const float lse2 = l[a] == 0.f ? neg_inf() : m[a] + log2f(l[a]);
            const int r = wid * 4 + a, hq = h * p.G + (pc.t * MI + r - tok[a] * p.G);
            const size_t orow = ((size_t)pc.w * p.Hq + hq) * p.S + tok[a];
            if (whole) {
#pragma unroll
                for (int c = 0; c < VC; ++c) static_cast<float*>(p.out)[orow * E + lane * VC + c] = o[a][c] * inv;
                if (p.lse_out && lane == 0) p.lse_out[orow] = lse2 * kLn2;
            } else {
#pragma unroll
                for (int c = 0; c < VC; ++c) p.part_o[(slot * MI + r) * E + lane * VC + c] = o[a][c] * inv;
                if (lane == 0) p.part_lse[slot * MI + r] = lse2;
            }
        }
    }
}

// ---- merge ----------------------------------------------------------------------------
// Rows of items that more than one group worked on: the log-sum-exp combination of their
// partials, in group order.  E / 4 lanes per row, two rows each.  Everything but the partials
// is known before the attention kernel ends (the prep kernel has ended when this one is
// launched); after the wait the sums and columns of up to kMergeAhead partials are read in one
// round trip.  Four at a time leave 48 registers and more resident blocks: 32 sequences 89 us, with
// eight (66 registers) 94; one sequence in 33 parts 30 and 29.  A call whose error word is set gets
// NaN in every output.
//
// 16-bit types: the attention kernel has taken infinities and NaN out of values that some tokens see and
// others do not (tree_tc.cu).  Such an element decides its output whatever the rest is, so it is
// added to the finished row of who sees it.
constexpr int kMergeAhead = 4;

template <class T> __device__ __forceinline__ void load_quad(const T* src, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2*>(src);
    const T* y = reinterpret_cast<const T*>(&x);
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = Elem<T>::to_f(y[c]);
}

template <class T, int E>
__global__ void __launch_bounds__(256, 5) tree_merge_kernel(TreeParams p) {
    constexpr int TPR = E / 4, RPB = 256 / TPR;  // threads per row, rows per block
    const int tid = threadIdx.x, lane = tid & 31;
    const int item = blockIdx.x, h = item % p.Hkv, t = item / p.Hkv % p.nt, w = item / p.Hkv / p.nt;
    const float nan = __int_as_float(0x7fc00000);
    // the groups that hold the item's first and last window
    long long total = 0, before = 0;
    for (int x = lane; x < p.W; x += 32) {
        const int n = __ldcg(p.nwin + x);
        total += n;
        if (x < w) before += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    const int nw = __ldcg(p.nwin + w);
    const SplitRange range(total * p.nt, p);
    const long long us = before * p.nt + (long long)t * nw;
    const int g0 = range.group_of(us), g1 = range.group_of(us + nw - 1);
    const int e = tid % TPR * 4;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int2 flags = __ldcg(reinterpret_cast<const int2*>(p.header + 2));
    const bool failed = flags.y != 0;
    // a value of the sequence and KV head has to be added
    const bool odd = sizeof(T) == 2 && flags.x && __ldcg(p.odd_any + w * p.Hkv + h);
    if (g0 == g1 && !failed && !odd) return;
    for (int i = blockIdx.y * RPB + tid / TPR; i < p.mi && (g0 != g1 || failed); i += gridDim.y * RPB) {
        const int r = t * p.mi + i;
        if (r >= p.rows) break;
        const int s = r / p.G, hq = h * p.G + r - s * p.G;
        const size_t orow = ((size_t)w * p.Hq + hq) * p.S + s;
        T* op = static_cast<T*>(p.out) + orow * E + e;
        if (failed) {
            store_quad<T>(op, nan, nan, nan, nan);
            if (p.lse_out && e == 0) p.lse_out[orow] = nan;
            continue;
        }
        float m = neg_inf(), den = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
        for (int g = g0; g <= g1; g += kMergeAhead) {
            float x[kMergeAhead];
            float4 v[kMergeAhead];
#pragma unroll
            for (int k = 0; k < kMergeAhead; ++k) {
                const int gg = g + k;
                const size_t at = (((size_t)gg * p.Hkv + h) * 2 + (gg == g0 ? 1 : 0)) * p.mi + i;
                x[k] = neg_inf();
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (g + k <= g1) {
                    x[k] = __ldcg(p.part_lse + at);
                    v[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * E + e));
                }
            }
            float mx = m;
            bool bad = false;  // fmaxf drops a NaN, the result must not
#pragma unroll
            for (int k = 0; k < kMergeAhead; ++k) {
                mx = fmaxf(mx, x[k]);
                bad |= x[k] != x[k];
            }
            const float mu = mx == neg_inf() ? 0.f : mx, alpha = fast_exp2(m - mu);
            m = mx;
            den = bad ? nan : den * alpha;
#pragma unroll
            for (int c = 0; c < 4; ++c) a[c] *= alpha;
#pragma unroll
            for (int k = 0; k < kMergeAhead; ++k) {
                if (x[k] == neg_inf()) continue;  // an empty part adds nothing
                const float f = fast_exp2(x[k] - mu);
                den += f;
                a[0] = fmaf(f, v[k].x, a[0]);
                a[1] = fmaf(f, v[k].y, a[1]);
                a[2] = fmaf(f, v[k].z, a[2]);
                a[3] = fmaf(f, v[k].w, a[3]);
            }
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        store_quad<T>(op, a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
        if (p.lse_out && e == 0) p.lse_out[orow] = den == 0.f ? neg_inf() : (m + log2f(den)) * kLn2;
    }
    // ---- infinities and NaN, added to the finished rows ----
    if constexpr (sizeof(T) == 2)
        if (odd && !failed)
#pragma unroll 1
            for (int i = blockIdx.y * RPB + tid / TPR; i < p.mi && t * p.mi + i < p.rows; i += gridDim.y * RPB) {
                const int r = t * p.mi + i, s = r / p.G;
                T* op = static_cast<T*>(p.out) + (((size_t)w * p.Hq + h * p.G + r - s * p.G) * p.S + s) * E + e;
                float a[4];
                load_quad(op, a);
                auto add = [&](const T* v) {
                    float x[4];
                    load_quad(v + e, x);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (!isfinite(x[c])) a[c] += x[c];
                };
                const size_t drafts = ((size_t)w * p.Hkv + h) * p.S;
                const uint32_t* anc = p.anc + ((size_t)w * p.S + s) * p.SW;
#pragma unroll 1
                for (int j = 0; j <= s; ++j)
                    if (__ldcg(p.odd + drafts + j) && (__ldcg(anc + (j >> 5)) >> (j & 31) & 1u)) add(static_cast<const T*>(p.dv) + (drafts + j) * E);
#pragma unroll 1
                for (int f = 0; f < p.F; ++f) {
                    const int2 span = __ldcg(p.span + (size_t)w * p.F + f);
                    if (span.y >= 0) continue;  // every token sees the same keys of the turn
                    // those of the windows that were looked through, and a few before them: what the row
                    // has already is the same when it counts twice
                    const int first = span.y & 0x7fffffff, lim = __ldcg(p.lim + ((size_t)f * p.W + w) * p.S + s);
#pragma unroll 1
                    for (int l = max(0, __ldcg(p.same + (size_t)w * p.F + f) - p.kt); l < lim; ++l) {
                        const int pos = first + l, page = __ldg(p.bt + (size_t)w * p.maxb + pos / p.BS);
                        if (page >= 0 && page < p.NB) add(static_cast<const T*>(p.v) + (((size_t)page * p.BS + pos % p.BS) * p.Hkv + h) * E);
                    }
                }
                store_quad<T>(op, a[0], a[1], a[2], a[3]);
            }
}

// ---------------------------------------------------------------------------------------
constexpr int kTreeMaxTokens = 1024;

template <int E> static TreeKernel simt_kernel() {
    TreeKernel k{};
    k.fn = (const void*)&tree_simt_kernel<E>;
    k.threads = SimtCfg<E>::THREADS;
    k.kt = SimtCfg<E>::KT;
    k.mi = SimtCfg<E>::MI;
    k.smem = SimtCfg<E>::SMEM;
    k.least = 1;  // 1024 keys, 4 tokens: 29 us, with 2 and 4 windows 33 and 45: a window takes it 4 us
    k.ctas = E == 256 ? 1 : E == 128 ? 2 : 4;  // by their shared memory: 170, 90, 49 KB
    return k;
}
static TreeKernel tree_pick(const dvattn_tree_args* a) {
    if (a->dtype != DVATTN_FLOAT32) return tree_tc_pick(a->dtype, a->E, a->S * (a->Hq / a->Hkv));
    return a->E == 64 ? simt_kernel<64>() : a->E == 128 ? simt_kernel<128>() : simt_kernel<256>();
}

// DVATTN_TEST_STALL_TILE=<i>: tests only (see the decode launcher); read once per process.
static int tree_stall_hook() {
    static const int t = [] {
        const char* e = getenv("DVATTN_TEST_STALL_TILE");
        return e && *e ? atoi(e) : -1;
    }();
    return t;
}

// Blocks of a sequence that rotate its drafted keys and its queries, and (16-bit types) copy its drafted values.
static long long tree_prep_blocks(const dvattn_tree_args* a) {
    const long long per = (long long)a->S * (a->E * (a->dtype == DVATTN_FLOAT32 ? 4 : 2) / 16);
    const long long values = a->dtype == DVATTN_FLOAT32 ? 0 : a->Hkv * per;
    return (((long long)a->Hq + a->Hkv) * per + kPrepChunks - 1) / kPrepChunks + (values + kPrepChunks - 1) / kPrepChunks;
}

static int tree_validate(const dvattn_tree_args* a) {
    if (!a) return DVATTN_ERR_INVALID_ARGUMENT;
    dvattn_paged_args v{};  // the shape rules of the paged attention
    v.dtype = a->dtype; v.F = a->F; v.W = a->W; v.Hq = a->Hq; v.Hkv = a->Hkv; v.E = a->E; v.Ev = a->Ev; v.S = a->S;
    v.R = a->R; v.block_size = a->block_size; v.max_blocks_per_seq = a->max_blocks_per_seq; v.num_blocks = a->num_blocks;
    const int st = decode_validate(&v);
    if (st != DVATTN_OK) return st;
    if (a->F < 1) return DVATTN_ERR_INVALID_ARGUMENT;  // the drafted tokens belong to the last turn
    if (a->S > kTreeMaxTokens) return DVATTN_ERR_UNSUPPORTED;
    // grid limits: sequences are the prep grid's x, row blocks its y; items are the merge grid's x
    const long long rows = (long long)a->S * (a->Hq / a->Hkv);
    if ((long long)a->F * a->W * a->Hq * a->S > 0x7fffffffLL || tree_prep_blocks(a) > 65534 ||
        (long long)a->W * a->Hkv * ((rows + 31) / 32) > 0x7fffffffLL)
        return DVATTN_ERR_UNSUPPORTED;
    return DVATTN_OK;
}

struct TreeLayout {
    size_t nwin, span, anc, lim, same, odd, odd_any, dkr, dvr, qr, po, pl, total;
    int groups, sw, nt;
};

static int tree_layout(const dvattn_tree_args* a, const TreeKernel& k, TreeLayout& L) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return DVATTN_ERR_CUDA;
    if (cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem) != cudaSuccess ||
        cudaFuncSetAttribute(k.fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess)
        return DVATTN_ERR_CUDA;
    L.groups = sms * k.ctas / a->Hkv;
    if (L.groups < 1) L.groups = 1;
    L.sw = (a->S + 127) / 128 * 4;
    L.nt = (int)(((long long)a->S * (a->Hq / a->Hkv) + k.mi - 1) / k.mi);
    const size_t ctas = (size_t)L.groups * a->Hkv, esz = a->dtype == DVATTN_FLOAT32 ? 4 : 2;
    size_t at = 256;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    L.nwin = take(4 * (size_t)a->W);
    L.span = take(8 * (size_t)a->W * a->F);
    L.anc = take(4 * (size_t)a->W * a->S * L.sw);
    L.lim = take(4 * (size_t)a->F * a->W * a->S);
    L.same = take(4 * (size_t)a->W * a->F);
    L.odd = take((size_t)a->W * a->Hkv * a->S);
    L.odd_any = take(4 * (size_t)a->W * a->Hkv);
    L.qr = take(esz * (size_t)a->F * a->W * a->Hq * a->S * a->E);
    L.dkr = take(esz * (size_t)a->W * a->Hkv * a->S * a->E);
    L.dvr = take(esz == 2 ? esz * (size_t)a->W * a->Hkv * a->S * a->E : 0);
    L.po = take(4 * ctas * 2 * k.mi * a->E);
    L.pl = take(4 * ctas * 2 * k.mi);
    L.total = at;
    return DVATTN_OK;
}

size_t tree_workspace_size(const dvattn_tree_args* a) {
    if (tree_validate(a) != DVATTN_OK || (long long)a->W * a->S == 0 || a->Hq == 0) return 0;
    TreeLayout L;
    return tree_layout(a, tree_pick(a), L) == DVATTN_OK ? L.total : 0;
}

static bool aligned16(const void* x) { return !(reinterpret_cast<uintptr_t>(x) & 15); }

template <class T> static const void* merge_fn(int E) {
    return E == 64 ? (const void*)&tree_merge_kernel<T, 64> : E == 128 ? (const void*)&tree_merge_kernel<T, 128>
                                                                      : (const void*)&tree_merge_kernel<T, 256>;
}

int tree_launch(const dvattn_tree_args* a, void* workspace, size_t wbytes, cudaStream_t stream) {
    int st = tree_validate(a);
    if (st != DVATTN_OK) return st;
    if ((long long)a->W * a->S == 0 || a->Hq == 0) return DVATTN_OK;
    if (!a->out || !a->queries || !a->parents || !a->locations || !a->fragment_lengths || !a->draft_keys || !a->draft_values ||
        (a->R > 0 && (!a->cosines || !a->sines)))
        return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->max_blocks_per_seq > 0 && a->num_blocks > 0 && (!a->k_cache || !a->v_cache || !a->block_tables))
        return DVATTN_ERR_INVALID_ARGUMENT;
    for (const void* x : {a->queries, a->k_cache, a->v_cache, a->draft_keys, a->draft_values, (const void*)a->out})
        if (!aligned16(x)) return DVATTN_ERR_INVALID_ARGUMENT;
    const TreeKernel k = tree_pick(a);
    TreeLayout L;
    if ((st = tree_layout(a, k, L)) != DVATTN_OK) return st;
    if (!workspace || wbytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return DVATTN_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    TreeParams p{};
    p.F = a->F; p.W = a->W; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv; p.S = a->S; p.R = a->R;
    p.rows = p.S * p.G;
    p.rot_vec = rotate_vec(a->R, a->cosines, a->sines);
    p.tail = a->S; p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.NB = a->num_blocks;
    const long long cap = (long long)a->max_blocks_per_seq * a->block_size;
    p.cap = a->num_blocks <= 0 ? 0 : cap > kMostPositions ? kMostPositions : (int)cap;
    p.SW = L.sw; p.kt = k.kt; p.mi = k.mi; p.nt = L.nt; p.groups = L.groups; p.least = k.least;
    p.scale_log2 = a->scale * kLog2e;
    p.out = a->out; p.lse_out = a->lse_out; p.q = a->queries; p.cos = a->cosines; p.sin = a->sines;
    p.loc = a->locations; p.L = a->fragment_lengths; p.parents = a->parents;
    p.k = a->k_cache ? a->k_cache : a->draft_keys; p.v = a->v_cache ? a->v_cache : a->draft_values;
    p.bt = a->block_tables; p.dk = a->draft_keys; p.dv = a->draft_values;
    p.stall_tile = tree_stall_hook();
    p.header = reinterpret_cast<int*>(ws);
    p.nwin = reinterpret_cast<int*>(ws + L.nwin);
    p.span = reinterpret_cast<int2*>(ws + L.span);
    p.lim = reinterpret_cast<int*>(ws + L.lim);
    p.same = reinterpret_cast<int*>(ws + L.same);
    p.odd = reinterpret_cast<uint8_t*>(ws + L.odd);
    p.odd_any = reinterpret_cast<int*>(ws + L.odd_any);
    p.qr = ws + L.qr;
    p.anc = reinterpret_cast<uint32_t*>(ws + L.anc);
    p.dkr = ws + L.dkr;
    p.dvr = ws + L.dvr;
    p.part_o = reinterpret_cast<float*>(ws + L.po);
    p.part_lse = reinterpret_cast<float*>(ws + L.pl);

    alignas(64) TreeMaps maps;
    p.align = 1;
    if (a->dtype != DVATTN_FLOAT32 && !tree_tc_maps(p, a->dtype, a->E, maps)) return DVATTN_ERR_CUDA;
    const void* prep = a->dtype == DVATTN_FLOAT32   ? (const void*)&tree_prep_kernel<float>
                       : a->dtype == DVATTN_FLOAT16 ? (const void*)&tree_prep_kernel<__half> : (const void*)&tree_prep_kernel<__nv_bfloat16>;
    const void* merge = a->dtype == DVATTN_FLOAT32   ? merge_fn<float>(a->E)
                        : a->dtype == DVATTN_FLOAT16 ? merge_fn<__half>(a->E) : merge_fn<__nv_bfloat16>(a->E);
    int E = a->E;
    void* pargs[] = {&p, &E};
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = stream;
    cfg.gridDim = dim3(a->W, 1 + (unsigned)tree_prep_blocks(a));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 2 * sizeof(int) * (size_t)a->S;
    cudaError_t e = cudaLaunchKernelExC(&cfg, prep, pargs);
    cfg.gridDim = dim3((unsigned)(L.groups * a->Hkv));
    cfg.blockDim = dim3(k.threads);
    cfg.dynamicSmemBytes = k.smem;
    void* args[] = {&p, &maps};  // the CUDA-core and merge kernels take the first only
    if (e == cudaSuccess) e = cudaLaunchKernelExC(&cfg, k.fn, args);
    if (e == cudaSuccess) {
        const int rpb = 256 / (a->E / 4), rows_max = L.nt > 1 ? k.mi : a->S * p.G;
        cfg.gridDim = dim3((unsigned)((long long)a->W * L.nt * a->Hkv), (unsigned)((rows_max + 2 * rpb - 1) / (2 * rpb)));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelExC(&cfg, merge, args);
    }
    if (e != cudaSuccess) {
        if (getenv("DVATTN_DEBUG")) fprintf(stderr, "dvattn tree launch: %s\n", cudaGetErrorString(e));
        return DVATTN_ERR_CUDA;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
