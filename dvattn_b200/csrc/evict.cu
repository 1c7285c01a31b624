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
// One launch, a cluster of blocks per (w, h): the survivors (a radix selection with the keys in
// registers), the list of moves, the mass and origin of every position that no move touches, then
// the moves: K and V rows, mass and origin.
//
// Bound: few moves, the latency of the selection's dependent steps; many, HBM (each moved row is
// read and written once).  128 rows of 4128 tokens, up to 28 moves each: 16 us (24 with one block a
// row, a batch of one key a thread and the moves in a second launch); 64 rows of 9000 to 30000
// tokens thinned out to 4001, 213 MB: 65 us, 51% of HBM's copy rate (133 that way), of which the
// selection is about 25.
#include "decode.cuh"

#include <cstdio>
#include <cstdlib>

namespace dvb {

struct EvictParams {
    int W, Hkv, BS, maxb, sink, recent;
    int C;      // blocks per row
    int words;  // 32-bit words of a bitmap over a block's tokens
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
    int2* moves;      // workspace [W * Hkv][N / 2] {to, from}, logical positions
    uint32_t* maps;   // workspace [W * Hkv * C][2][words] unless smem_maps
};

constexpr int kSelThreads = 1024;
constexpr int kSelKeys = 16;  // keys of a thread in flight, and kept for the next pass where a chunk has no more
constexpr int kBins = 2048;
constexpr int kMoveBatch = 8;  // moves of a warp at a time, at most
constexpr int kMoveChunks = 4; // 16-byte chunks a lane loads before it stores

// Order of a mass as an unsigned integer: larger mass, larger key; -0 equals +0; NaN lowest.
__device__ __forceinline__ uint32_t mass_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix sum of one value per thread over the block, and the total.  `sh`: 32 values of
// this scan alone.
template <class V> __device__ __forceinline__ V block_scan(V v, V* sh, V& total) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    V incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 31) sh[wid] = incl;
    __syncthreads();
    V warps = sh[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V up = __shfl_up_sync(0xffffffffu, warps, o);
        if (lane >= o) warps += up;
    }
    total = __shfl_sync(0xffffffffu, warps, 31);
    const V before = __shfl_sync(0xffffffffu, warps, wid > 0 ? wid - 1 : 0);
    return (wid > 0 ? before : V(0)) + incl - v;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// two neighbouring words of another block's shared memory, at the same place as `own` of this one's
__device__ __forceinline__ int2 cluster_load(const int* own, uint32_t rank) {
    uint32_t a;
    int2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(own)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}

// A cluster of p.C blocks per row, each a chunk of its tokens.  The blocks exchange histograms and
// counts through distributed shared memory; each finds the same digits for itself.
__global__ void __launch_bounds__(kSelThreads) evict_kernel(EvictParams p) {
    static_assert(kSelThreads == 32 * 32 && kBins == 2 * kSelThreads, "block_scan; a thread scans two bins");
    extern __shared__ uint32_t dyn[];  // 2 bitmaps, if smem_maps
    __shared__ __align__(8) int hist[3][kBins];
    __shared__ int sh[4][32];
    __shared__ unsigned long long sh2[32];
    __shared__ __align__(8) int s_moves[2];  // holes and movers of the chunk
    __shared__ int s_digit[3], s_above[3];
    const int tid = threadIdx.x, lane = tid & 31;
    const unsigned C = p.C, rank = cluster_rank();
    const int row = blockIdx.x / C, w = row / p.Hkv;
    const float* mass = p.mass + (size_t)row * p.N;
    const long long start64 = __ldg(p.starts + w), len64 = __ldg(p.lengths + w);
    const long long lim = p.N < p.cap ? p.N : p.cap;  // positions that have a mass and a place in the table
    const int start = start64 < 0 || start64 > lim ? 0 : (int)start64;
    const int n = start64 < 0 || start64 >= lim || len64 <= 0 ? 0 : (int)(len64 < lim - start ? len64 : lim - start);
    const int keep = max(__ldg(p.keep + w), 0), kept = min(n, keep);
    const bool all = kept == n, none = kept == 0, choose = !all && !none;
    // the block's tokens: c0 + i for i < m
    const unsigned chunk = (((unsigned)n + C - 1) / C + 31u) & ~31u;
    const int c0 = (int)min(rank * chunk, (unsigned)n), m = (int)min(chunk, (unsigned)(n - c0));
    // a thread's keys of kSelKeys strides of the block from i0 on; the loads are in flight together,
    // and a chunk of one such batch is read once for all passes
    uint32_t key[kSelKeys];
    int loaded = -1;
    auto sweep = [&](auto&& each) {  // each(i, key) for every i below m rounded up to whole warps
        for (int i0 = 0; i0 < m; i0 += kSelKeys * kSelThreads) {
            if (choose && loaded != i0) {
                loaded = i0;
                float x[kSelKeys];
#pragma unroll
                for (int u = 0; u < kSelKeys; ++u) {
                    const int i = i0 + u * kSelThreads + tid;
                    x[u] = i < m ? mass[start + c0 + i] : 0.f;
                }
#pragma unroll
                for (int u = 0; u < kSelKeys; ++u) {
                    const int i = c0 + i0 + u * kSelThreads + tid;
                    key[u] = i < p.sink || i >= n - p.recent ? 0xffffffffu : mass_key(x[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < kSelKeys; ++u) {
                const int i = i0 + u * kSelThreads + tid;
                if (i - lane >= m) break;
                each(i, key[u]);
            }
        }
    };
    // ---- the kept-th largest key, 11 + 11 + 10 bits at a time ----
    uint32_t prefix = 0;
    int need = kept;       // survivors still to be found among the keys that share the prefix
    int ties_before = 0;   // keys equal to it in the chunks before
    if (choose) {
        for (int i = tid; i < 3 * kBins; i += kSelThreads) hist[0][i] = 0;
        __syncthreads();
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            sweep([&](int i, uint32_t k) {
                if (i < m && (pass == 0 || (k >> (shift + bits)) == (prefix >> (shift + bits))))
                    atomicAdd(&hist[pass][(k >> shift) & ((1u << bits) - 1)], 1);
            });
            cluster_sync();
            // bins from the top down: thread t holds bins top - 2t, top - 2t - 1
            const int b = kBins - 1 - 2 * tid;
            int k0 = 0, k1 = 0, total;
            for (unsigned r = 0; r < C; ++r) {
                const int2 x = cluster_load(&hist[pass][b - 1], r);
                k0 += x.y, k1 += x.x;
            }
            const int above = block_scan(k0 + k1, sh[pass], total);
            if (above < need && need <= above + k0) s_digit[pass] = b, s_above[pass] = above;
            if (above + k0 < need && need <= above + k0 + k1) s_digit[pass] = b - 1, s_above[pass] = above + k0;
            __syncthreads();
            prefix |= (uint32_t)s_digit[pass] << shift;
            need -= s_above[pass];
        }
        const int d = s_digit[2];
        for (unsigned r = 0; r < rank; ++r) {
            const int2 x = cluster_load(&hist[2][d & ~1], r);
            ties_before += d & 1 ? x.y : x.x;
        }
    }
    // survivors: keys above `prefix`, and the first `need` keys equal to it
    uint32_t* m_keep = p.smem_maps ? dyn : p.maps + (size_t)blockIdx.x * 2 * p.words;
    uint32_t* m_tie = m_keep + p.words;
    const int words = (m + 31) / 32;
    sweep([&](int i, uint32_t k) {
        const unsigned a = __ballot_sync(0xffffffffu, i < m && (all || (choose && k > prefix)));
        const unsigned t = __ballot_sync(0xffffffffu, i < m && choose && k == prefix);
        if (lane == 0) m_keep[i >> 5] = a, m_tie[i >> 5] = t;
    });
    __syncthreads();
    // a thread owns `per` words: first the ties, then holes and movers
    const int per = (words + kSelThreads - 1) / kSelThreads, w0 = min(tid * per, words), w1 = min(w0 + per, words);
    {
        int c = 0, total;
        for (int x = w0; x < w1; ++x) c += __popc(m_tie[x]);
        int left = need - ties_before - block_scan(c, sh[3], total);
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
        const int d = kept - c0 - 32 * x;
        return d <= 0 ? 0u : d >= 32 ? 0xffffffffu : (1u << d) - 1;
    };
    auto present = [&](int x) { return m - 32 * x >= 32 ? 0xffffffffu : (1u << (m - 32 * x)) - 1; };  // x < words
    int nh = 0, nm = 0;
    for (int x = w0; x < w1; ++x) {
        const uint32_t k = m_keep[x], f = below(x);
        nh += __popc(~k & f & present(x));
        nm += __popc(k & ~f);
    }
    unsigned long long total;
    const unsigned long long at = block_scan((unsigned long long)nh << 32 | (unsigned)nm, sh2, total);
    if (tid == 0) s_moves[0] = (int)(total >> 32), s_moves[1] = (int)(total & 0xffffffffu);
    cluster_sync();  // and m_keep is complete
    int ih = (int)(at >> 32), im = (int)(at & 0xffffffffu), moved = 0;
    for (unsigned r = 0; r < C; ++r) {
        const int2 x = cluster_load(s_moves, r);
        moved += x.x;
        if (r < rank) ih += x.x, im += x.y;
    }
    int2* mv = p.moves + (size_t)row * (p.N / 2);
    for (int x = w0; x < w1; ++x) {
        const uint32_t k = m_keep[x], f = below(x);
        for (uint32_t hole = ~k & f & present(x); hole; hole &= hole - 1) mv[ih++].x = start + c0 + 32 * x + __ffs(hole) - 1;
        for (uint32_t mover = k & ~f; mover; mover &= mover - 1) mv[im++].y = start + c0 + 32 * x + __ffs(mover) - 1;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // its part of the list is written
    // ---- mass and origin of what no move touches; in place, most of the mass stays ----
    float* mout = p.mass_out + (size_t)row * p.N;
    int* src = p.source ? p.source + (size_t)row * p.N : nullptr;
    const bool in_place = mout == mass;
    constexpr int U = 8;
    for (int i0 = tid; i0 < m; i0 += U * kSelThreads) {
        const int q0 = start + c0 + i0;
        float x[U];
        int what[U];  // 0: a move's, 1: stays, 2: evicted
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kSelThreads;
            what[u] = 0;
            if (i >= m) break;
            const bool k = m_keep[i >> 5] >> (i & 31) & 1u;
            what[u] = c0 + i < kept ? (k ? 1 : 0) : (k ? 0 : 2);
            x[u] = what[u] == 1 && !in_place ? mass[q0 + u * kSelThreads] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * kSelThreads >= m) break;
            const int q = q0 + u * kSelThreads;
            if (what[u] == 2 || (what[u] == 1 && !in_place)) mout[q] = x[u];
            if (src && what[u] != 0) src[q] = what[u] == 2 ? -1 : q;
        }
    }
    if (src || !in_place) {  // positions outside the tokens
        for (long long i = (long long)rank * kSelThreads + tid; i < p.N - n; i += C * kSelThreads) {
            const long long q = i < start ? i : i + n;
            if (!in_place) mout[q] = mass[q];
            if (src) src[q] = (int)q;
        }
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    // ---- the moves: a warp takes up to kMoveBatch; a lane each reads them, finds their rows and
    // moves their mass, then the lanes copy the 16-byte chunks of their K and V rows, kMoveChunks
    // loads in flight ----
    const int h = row - w * p.Hkv, warps = C * (kSelThreads / 32), cpm = p.ck + p.cv;
    const int batch = min(kMoveBatch, (moved + warps - 1) / warps);
    const int* bt = p.bt + (size_t)w * p.maxb;
    for (int i0 = ((int)rank * (kSelThreads / 32) + (tid >> 5)) * batch; i0 < moved; i0 += warps * batch) {
        const int mine = min(batch, moved - i0);
        long long to = -1, from = 0;
        if (lane < mine) {
            const int2 x = __ldcg(mv + i0 + lane);
            const int pd = __ldg(bt + x.x / p.BS), ps = __ldg(bt + x.y / p.BS);
            if (pd >= 0 && pd < p.NB && ps >= 0 && ps < p.NB) {
                to = ((long long)pd * p.BS + x.x % p.BS) * p.Hkv + h;
                from = ((long long)ps * p.BS + x.y % p.BS) * p.Hkv + h;
            }
            mout[x.x] = __ldcg(mass + x.y);  // nobody else reads or writes either place
            mout[x.y] = 0.f;
            if (src) src[x.x] = x.y, src[x.y] = -1;
        }
        int y = lane / cpm, c = lane - y * cpm;  // move and chunk
        while (__any_sync(0xffffffffu, y < mine)) {
            uint4 v[kMoveChunks];
            uint4* dst[kMoveChunks];
#pragma unroll
            for (int u = 0; u < kMoveChunks; ++u) {
                const long long d = __shfl_sync(0xffffffffu, to, y & (kMoveBatch - 1)), s = __shfl_sync(0xffffffffu, from, y & (kMoveBatch - 1));
                dst[u] = nullptr;
                if (y < mine && d >= 0) {
                    const bool k = c < p.ck;
                    const uint4* base = static_cast<const uint4*>(k ? p.k : p.v) + (k ? c : c - p.ck);
                    dst[u] = const_cast<uint4*>(base) + d * (k ? p.ck : p.cv);
                    v[u] = __ldcg(base + s * (k ? p.ck : p.cv));
                }
                for (c += 32; c >= cpm; c -= cpm) ++y;
            }
#pragma unroll
            for (int u = 0; u < kMoveChunks; ++u)
                if (dst[u]) *dst[u] = v[u];
        }
    }
}

// ---------------------------------------------------------------------------------------
// Up to this many bytes of bitmaps a block keeps them in shared memory (chunks of 65536 tokens); longer chunks have them in the workspace.
constexpr int kMapSmem = 16 * 1024;
constexpr int kMaxCluster = 8;  // portable
constexpr int kChunk = 4096;

static int evict_validate(const dvattn_evict_args* a) {
    if (!a) return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->dtype < 0 || a->dtype > 2) return DVATTN_ERR_UNSUPPORTED;
    if (a->W < 0 || a->Hkv <= 0 || a->E <= 0 || a->Ev <= 0 || a->block_size <= 0 || a->max_blocks_per_seq < 0 || a->num_blocks < 0 ||
        a->positions < 0 || a->sink < 0 || a->recent < 0)
        return DVATTN_ERR_INVALID_ARGUMENT;
    const int esz = a->dtype == DVATTN_FLOAT32 ? 4 : 2;
    if ((a->E * esz) % 16 || (a->Ev * esz) % 16) return DVATTN_ERR_UNSUPPORTED;
    if (a->positions > 0x7fff0000LL || (long long)a->max_blocks_per_seq * a->block_size > 0x7fffffffLL ||
        (long long)a->W * a->Hkv > 65535)
        return DVATTN_ERR_UNSUPPORTED;
    return DVATTN_OK;
}
static bool evict_nothing(const dvattn_evict_args* a) { return a->W == 0 || a->positions == 0; }

struct EvictLayout {
    size_t moves, maps, total;
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
    L.moves = take(8 * rows * (size_t)(a->positions / 2));
    // for any number of blocks per row: a chunk's last word may be rounded up twice
    L.maps = take(8LL * ((a->positions + 31) / 32) <= kMapSmem ? 0 : 8 * rows * (size_t)(a->positions / 32 + 2 * kMaxCluster));
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
    p.ck = a->E * esz / 16; p.cv = a->Ev * esz / 16;
    p.k = a->k_cache; p.v = a->v_cache; p.mass = a->mass; p.mass_out = a->mass_out; p.source = a->source;
    p.bt = a->block_tables; p.starts = a->starts; p.lengths = a->lengths; p.keep = a->keep;
    p.moves = reinterpret_cast<int2*>(ws + L.moves);
    p.maps = reinterpret_cast<uint32_t*>(ws + L.maps);
    const int rows = a->W * a->Hkv;
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return DVATTN_ERR_CUDA;
    // Blocks per row: more while a chunk has more than kChunk positions and every block has an SM of
    // its own.  One block's passes are bound by its SM's instructions: 64 rows of up to 30000 tokens
    // take 105 us with one block each, 68 with two; 8 rows 97 with one, 55 with two, 35 with eight.
    p.C = 1;
    while (p.C < kMaxCluster && a->positions > (long long)p.C * kChunk && 2LL * p.C * rows <= sms) p.C *= 2;
    p.words = (int)(((a->positions + p.C - 1) / p.C + 31) / 32);
    p.smem_maps = 8LL * p.words <= kMapSmem;
    void* args[] = {&p};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = stream;
    cfg.gridDim = dim3(rows * p.C);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = p.smem_maps ? 8 * (size_t)p.words : 0;
    const cudaError_t e = cudaLaunchKernelExC(&cfg, (const void*)&evict_kernel, args);
    if (e != cudaSuccess) {
        if (getenv("DVATTN_DEBUG")) fprintf(stderr, "dvattn evict launch: %s\n", cudaGetErrorString(e));
        return DVATTN_ERR_CUDA;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
