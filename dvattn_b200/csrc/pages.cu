// Block tables and slot maps from request lengths, on the GPU: pages taken from a free list (a stack) for the
// positions that a step's new tokens fall on, and pages given back.
//
// Both are a counting problem: of the entries looked at, in the order of (sequence, entry), the i-th that
// wants a page (that gives one back) meets the i-th free page.  One cluster of 8 blocks: a warp has a run of
// sequences, or where there are fewer sequences than warps a part of one's entries; the warps' counts are
// added up through shared memory and the clusters' distributed shared memory; then the same walk moves the
// pages.  A launch of its own writes long slot maps, with the whole GPU.
//
// Bound: the launch, the cluster's barriers, and the walks' instructions on 8 SMs.  So a walk over long rows (from 32
// entries a sequence on average, or one sequence's) goes row by row, 32 entries a load, and only short rows are packed 32 to a
// load with a search for each entry's owner; and the second walk ends behind the warp's last entry that moves.  Released
// and assigned, B200, replayed from a graph: 256 sequences with tables of 2001 pages, one token each, 26.7 us (48.5 with the search
// alone, of which the release's look at 512,256 entries took 39 and takes 11.6; calls by themselves 30.7); 48 prompts of up to 32,000
// tokens 34 us (91; by themselves 41.0).  A cluster of 16 blocks takes a tenth less but may not be launchable.
#include "decode.cuh"

#include <cooperative_groups.h>

namespace dvb {

namespace {

namespace cg = cooperative_groups;

constexpr int kBlocks = 8, kThreads = 1024, kWarps = kThreads / 32;
constexpr int kAhead = 8, kRowAhead = 16;  // entries a lane has in flight: of several rows, of one
constexpr int kAll = 0x7fffffff;
constexpr int kLongRows = 32 * 32;         // entries of 32 sequences from which a walk goes row by row
constexpr long long kSlotsHere = 1 << 15;  // a slot map up to this size is written by the cluster

struct PageParams {
    int W, BS, maxb, size, n;
    int per, parts;  // sequences of a warp, or warps of a sequence
    int* bt;
    int* free_pages;
    int* count;
    const int* starts;
    const int* counts;
    int* granted;
    long long* slots;  // written here; null: not, or by a launch of its own
};

// A chunk of up to 32 sequences, one per lane: entries [first, first + m) of its row are looked at.
struct Chunk {
    int w, first, m, upto;  // upto: entries of the lanes up to this one
    int all;
    bool bad;
    int count;
};
// part of `parts`: of its entries that much.
template <bool ASSIGN> __device__ __forceinline__ Chunk chunk_of(const PageParams& p, int w0, int w1, int part, int parts, int lane) {
    Chunk c;
    c.w = w0 + lane;
    c.first = c.m = c.count = 0;
    c.bad = false;
    if (c.w < w1) {
        const int s = __ldg(p.starts + c.w);
        if (ASSIGN) {
            c.count = max(__ldg(p.counts + c.w), 0);
            c.bad = s < 0 || (long long)s + c.count > (long long)p.maxb * p.BS;
            if (c.count > 0 && !c.bad) {
                c.first = s / p.BS;
                c.m = (s + c.count - 1) / p.BS - c.first + 1;
            }
        } else {
            c.first = s > 0 ? (int)min(((long long)s + p.BS - 1) / p.BS, (long long)p.maxb) : 0;
            c.m = p.maxb - c.first;
        }
    }
    if (parts > 1) {
        const int m0 = (int)((long long)c.m * part / parts), m1 = (int)((long long)c.m * (part + 1) / parts);
        c.first += m0, c.m = m1 - m0;
    }
    c.upto = c.m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, c.upto, o);
        if (lane >= o) c.upto += x;
    }
    c.all = __shfl_sync(0xffffffffu, c.upto, 31);
    return c;
}

// Calls f(mask of the lanes whose entry wants or gives, own entry's place, its value, owner lane, base, n) for every
// n <= 32 entries from `base` of the chunk, by the whole warp, those from `limit` on left out or not; place, value and owner are those of lanes below n.
template <bool ASSIGN, class F> __device__ __forceinline__ void each(const PageParams& p, const Chunk& c, int lane, int limit, F f) {
    if (c.all >= kLongRows || c.all > 0 && c.all == __shfl_sync(0xffffffffu, c.m, 0)) {  // long rows, or one sequence's
        for (int k = 0; k < 32; ++k) {
            const int m = __shfl_sync(0xffffffffu, c.m, k);
            if (m == 0) continue;
            const int start = __shfl_sync(0xffffffffu, c.upto, k) - m;
            const long long row = (long long)__shfl_sync(0xffffffffu, c.w, k) * p.maxb + __shfl_sync(0xffffffffu, c.first, k);
            for (int i0 = 0; i0 < m && start + i0 < limit; i0 += 32 * kRowAhead) {
                int val[kRowAhead];
#pragma unroll
                for (int u = 0; u < kRowAhead; ++u) {
                    const int i = i0 + 32 * u + lane;
                    val[u] = i < m ? __ldcg(p.bt + row + i) : (ASSIGN ? 0 : -1);
                }
#pragma unroll
                for (int u = 0; u < kRowAhead; ++u)
                    if (i0 + 32 * u < m)
                        f(__ballot_sync(0xffffffffu, ASSIGN ? val[u] < 0 : val[u] >= 0), row + i0 + 32 * u + lane, val[u], k, start + i0 + 32 * u, min(m - i0 - 32 * u, 32));
            }
        }
        return;
    }
    for (int base = 0; base < c.all && base < limit; base += 32 * kAhead) {
        long long at[kAhead];
        int own[kAhead], val[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = base + 32 * u + lane;
            int k = 0;  // lanes whose entries all lie in front
#pragma unroll
            for (int step = 16; step > 0; step >>= 1)
                if (__shfl_sync(0xffffffffu, c.upto, k + step - 1) <= i) k += step;
            own[u] = k;
            const int first = __shfl_sync(0xffffffffu, c.first, k), w = __shfl_sync(0xffffffffu, c.w, k);
            const int before = __shfl_sync(0xffffffffu, c.upto - c.m, k);
            at[u] = i < c.all ? (long long)w * p.maxb + first + (i - before) : -1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) val[u] = at[u] >= 0 ? __ldcg(p.bt + at[u]) : (ASSIGN ? 0 : -1);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) f(__ballot_sync(0xffffffffu, ASSIGN ? val[u] < 0 : val[u] >= 0), at[u], val[u], own[u], base + 32 * u, 32);
    }
}

// Entries of the lane's own sequence among the `mask` of entries from `base`.
__device__ __forceinline__ int own_part(const Chunk& c, unsigned mask, int base) {
    const int lo = max(c.upto - c.m - base, 0), hi = min(c.upto - base, 32);
    return hi > lo ? __popc(mask >> lo & (hi - lo == 32 ? 0xffffffffu : (1u << (hi - lo)) - 1)) : 0;
}

template <bool ASSIGN> __global__ void __cluster_dims__(kBlocks, 1, 1) __launch_bounds__(kThreads) pages_kernel(PageParams p) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_arrive();  // every block arrives once it runs: others write into its shared memory only after that
    __shared__ int warp_sum[kWarps];
    __shared__ int block_sum[2][kBlocks], block_used[kBlocks];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, rank = (int)cluster.block_rank(), me = rank * kWarps + wid;
    int w0, w1, part = 0, parts = p.parts;
    if (parts > 1) {
        w0 = min(me / parts, p.W), w1 = min(w0 + 1, p.W), part = me % parts;
    } else {
        w0 = (int)min((long long)me * p.per, (long long)p.W), w1 = (int)min((long long)me * p.per + p.per, (long long)p.W);
    }
    const int have = min(max(__ldcg(p.count), 0), p.size);  // pages on the stack
    // entries that want or give: this warp's, those in front of them, all; one exchange per buffer
    int mine = 0, before = 0, total = 0;
    int limit = 0;  // where a warp has one chunk: its last that want or give lie in front
    auto count = [&](int buffer) {
        int sum = 0;
        mine = 0, limit = 0;
        for (int w = w0; w < w1; w += 32) {
            const Chunk c = chunk_of<ASSIGN>(p, w, w1, part, parts, lane);
            each<ASSIGN>(p, c, lane, kAll, [&](unsigned mask, long long, int, int, int base, int) {
                mine += __popc(mask);
                if (mask) limit = base + 32;
            });
        }
        if (w1 - w0 > 32) limit = kAll;
        before = total = 0;
        if (lane == 0) warp_sum[wid] = mine;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) {
            if (i < wid) before += warp_sum[i];
            sum += warp_sum[i];
        }
        if (buffer == 0) cluster.barrier_wait();  // all blocks run (the first use of their shared memory)
        if (threadIdx.x < kBlocks) *cluster.map_shared_rank(&block_sum[buffer][rank], threadIdx.x) = sum;
        cluster.sync();
        for (int i = 0; i < kBlocks; ++i) {
            if (i < rank) before += block_sum[buffer][i];
            total += block_sum[buffer][i];
        }
    };
    count(0);
    int used = total;
    if (ASSIGN && total > have) {  // too few: the entries of the sequences that are served
        if (parts > 1) {           // whole sequences from here on
            parts = 1, part = 0;
            w0 = min(me, p.W), w1 = min(me + 1, p.W);
            count(1);
        }
        int top = 0, upto = before;
        for (int w = w0; w < w1; w += 32) {
            const Chunk c = chunk_of<ASSIGN>(p, w, w1, part, parts, lane);
            int need = 0;
            each<ASSIGN>(p, c, lane, kAll, [&](unsigned mask, long long, int, int, int base, int) { need += own_part(c, mask, base); });
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, need, o);
                if (lane >= o) need += x;
            }
            if (upto + need <= have) top = max(top, upto + need);
            upto += __shfl_sync(0xffffffffu, need, 31);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        __syncthreads();
        if (lane == 0) warp_sum[wid] = top;
        __syncthreads();
        for (int i = 0; i < kWarps; ++i) top = max(top, warp_sum[i]);
        if (threadIdx.x < kBlocks) *cluster.map_shared_rank(&block_used[rank], threadIdx.x) = top;
        cluster.sync();
        used = 0;
        for (int i = 0; i < kBlocks; ++i) used = max(used, block_used[i]);
    }
    const int room = ASSIGN ? 0 : min(total, p.size - have);  // pages that the list takes back
    // everyone has read the count: the clusters' barrier lies between
    if (rank == 0 && threadIdx.x == 0) *p.count = ASSIGN ? have - used : have + room;
    int upto = before;
    for (int w = w0; w < w1; w += 32) {
        const Chunk c = chunk_of<ASSIGN>(p, w, w1, part, parts, lane);
        bool given = true;
        if (ASSIGN) {
            int need = 0;
            if (total > have && mine > 0) each<ASSIGN>(p, c, lane, kAll, [&](unsigned mask, long long, int, int, int base, int) { need += own_part(c, mask, base); });
            int sums = need;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sums, o);
                if (lane >= o) sums += x;
            }
            given = !c.bad && (need == 0 || upto + sums <= have);
            if (c.w < w1 && part == 0) p.granted[c.w] = given ? c.count : 0;
        }
        if (mine == 0) continue;  // nothing moves here
        each<ASSIGN>(p, c, lane, limit, [&](unsigned mask, long long at, int val, int own, int, int) {
            const int i = upto + __popc(mask & ((1u << lane) - 1));
            const bool go = !ASSIGN || __shfl_sync(0xffffffffu, (int)given, own) != 0;
            if (mask >> lane & 1u) {
                if (ASSIGN) {
                    if (go) p.bt[at] = p.free_pages[have - used + i];
                } else if (i < room) {
                    p.free_pages[have + i] = val;
                    p.bt[at] = -1;
                }
            }
            upto += __popc(mask);
        });
    }
    cluster.sync();  // no block ends while another may still write into its shared memory; the tables are written
    if (ASSIGN && p.slots)
        for (int x = me * 32 + lane; x < p.W * p.n; x += kBlocks * kThreads) {
            const int w = x / p.n, i = x - w * p.n;
            long long slot = -1;
            if (i < __ldcg(p.granted + w)) {
                const int at = __ldg(p.starts + w) + i, page = __ldcg(p.bt + (size_t)w * p.maxb + at / p.BS);
                if (page >= 0) slot = (long long)page * p.BS + at % p.BS;
            }
            p.slots[x] = slot;
        }
}

// slots[w][i] from the tables and granted counts
__global__ void __launch_bounds__(256) slots_kernel(PageParams p) {
    const int w = blockIdx.y, n = __ldg(p.granted + w), s = __ldg(p.starts + w);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < p.n; i += (long long)gridDim.x * 256) {
        long long slot = -1;
        if (i < n) {
            const int at = s + (int)i, page = __ldg(p.bt + (size_t)w * p.maxb + at / p.BS);
            if (page >= 0) slot = (long long)page * p.BS + at % p.BS;
        }
        p.slots[(size_t)w * p.n + i] = slot;
    }
}

int pages_check(int W, int BS, int maxb, int size) {
    if (W < 0 || BS <= 0 || maxb < 0 || size < 0) return DVATTN_ERR_INVALID_ARGUMENT;
    // entries and positions are counted in 32 bits, entries by walks that step past the last one by up to 32 * kRowAhead
    if ((long long)W * maxb > 0x7fffffffLL - 2 * 32 * kRowAhead || (long long)maxb * BS > 0x7fffffffLL) return DVATTN_ERR_UNSUPPORTED;
    return DVATTN_OK;
}

}  // namespace

int assign_pages_launch(const dvattn_assign_args* a, cudaStream_t stream) {
    if (!a) return DVATTN_ERR_INVALID_ARGUMENT;
    const int st = pages_check(a->W, a->block_size, a->max_blocks_per_seq, a->free_size);
    if (st != DVATTN_OK) return st;
    if (a->n < 0) return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->W == 0) return DVATTN_OK;
    if (!a->free_count || !a->starts || !a->counts || !a->granted || (a->max_blocks_per_seq > 0 && !a->block_tables) || (a->free_size > 0 && !a->free_pages))
        return DVATTN_ERR_INVALID_ARGUMENT;
    // several warps read a sequence's start and count while one writes what it is granted
    for (const int* in : {a->starts, a->counts})
        if (a->granted < in + a->W && in < a->granted + a->W) return DVATTN_ERR_INVALID_ARGUMENT;
    PageParams p{};
    p.W = a->W; p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.size = a->free_size; p.n = a->n;
    p.per = (a->W + kBlocks * kWarps - 1) / (kBlocks * kWarps);
    p.parts = a->W < kBlocks * kWarps ? kBlocks * kWarps / a->W : 1;
    p.bt = a->block_tables; p.free_pages = const_cast<int*>(a->free_pages); p.count = a->free_count;
    p.starts = a->starts; p.counts = a->counts; p.granted = a->granted;
    const bool here = (long long)a->W * a->n <= kSlotsHere;
    p.slots = here && a->n > 0 ? a->slots : nullptr;
    pages_kernel<true><<<kBlocks, kThreads, 0, stream>>>(p);
    if (a->slots && a->n > 0 && !here) {
        p.slots = a->slots;
        for (int w = 0; w < a->W; w += 65535) {
            PageParams q = p;
            const int rows = a->W - w < 65535 ? a->W - w : 65535;
            q.granted += w, q.starts += w, q.bt += (size_t)w * p.maxb, q.slots += (size_t)w * p.n;
            slots_kernel<<<dim3((unsigned)((a->n + 1023) / 1024), (unsigned)rows), 256, 0, stream>>>(q);
        }
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

int release_pages_launch(const dvattn_release_args* a, cudaStream_t stream) {
    if (!a) return DVATTN_ERR_INVALID_ARGUMENT;
    const int st = pages_check(a->W, a->block_size, a->max_blocks_per_seq, a->free_size);
    if (st != DVATTN_OK) return st;
    if (a->W == 0 || a->max_blocks_per_seq == 0) return DVATTN_OK;
    if (!a->free_count || !a->keep || !a->block_tables || (a->free_size > 0 && !a->free_pages)) return DVATTN_ERR_INVALID_ARGUMENT;
    PageParams p{};
    p.W = a->W; p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.size = a->free_size;
    p.per = (a->W + kBlocks * kWarps - 1) / (kBlocks * kWarps);
    p.parts = a->W < kBlocks * kWarps ? kBlocks * kWarps / a->W : 1;
    p.bt = a->block_tables; p.free_pages = a->free_pages; p.count = a->free_count; p.starts = a->keep;
    pages_kernel<false><<<kBlocks, kThreads, 0, stream>>>(p);
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
