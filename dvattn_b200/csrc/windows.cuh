// The producer warp of the tensor-core kernels over the paged turns (tree_tc.cu, mass_tc.cu):
// fills a ring of swizzled [KT rows][E] tiles with the windows of the CTA's runs.
//
// Where pages and windows are whole numbers of boxes of 8 or more rows (page sizes that are
// multiples of 8), by TMA, one box per lane and 64-column panel; a box that holds no seen key
// loads zeros, other rows that nobody sees load what lies there.  Else rows are gathered with
// cp.async, and rows that nobody sees are zeros.
#pragma once

#include <type_traits>

#include "tma_host.cuh"
#include "turns.cuh"

namespace dvb {

// Rows of a TMA box: the largest power of two that divides the page size, at most a window; 0
// where it is below the 8 rows that the 128-byte swizzle repeats over, or a coordinate might not
// fit in 32 bits.
inline int window_box(int BS, int kt, long long NB) {
    int b = kt;
    while (BS % b) b >>= 1;
    return b < 8 || NB * BS > 0x7fffffffLL - 2 * (long long)BS ? 0 : b;
}

struct WindowSource {
    const void* cache;            // [NB][BS][Hkv][E]
    const void* tail;             // [W][Hkv][tail][E], or null where the split has no tail
    const CUtensorMap* map;
    const CUtensorMap* tail_map;
    const uint32_t* anc;          // [W][tail][SW]: a tail row without its own bit is not there
    int SW, h, Hkv;
    int box;                      // rows of a TMA box, 0: gathered
    int me, of;                   // this warp requests the windows me, me + of, ... of every run
    int stall;                    // test hook: this window never arrives; -1: off
    uint64_t policy;              // L2
};

// What is done to the tiles: nothing, or (the values of a drafted tree: tree_tc.cu) the windows of the runs
// for which in(run) is true, and of these those for which look(run, end) is true, `end` the key behind
// their last, are made finite, and found(run) is called where there was an infinity or NaN.  `raw`: an
// mbarrier per stage, on which the boxes of these windows land.
struct AsTheyAre {
    static constexpr bool always = true;
    static constexpr uint32_t raw = 0;
    bool leave;  // at the first run with RUN_MIXED
    __device__ __forceinline__ bool in(const SplitRun&) const { return false; }
    __device__ __forceinline__ bool look(const SplitRun&, int) const { return false; }
    __device__ __forceinline__ void found(const SplitRun&) const {}
};

// Where a producer is; a second call goes on from there.
struct Producer {
    SplitRun run;
    int nr, x, iw;  // runs taken, window of the run, tiles requested
    bool fresh;     // the run has not been opened
    int left;       // produce_windows returned at a mixed run of that many windows, 0: at the end
};

// Sum of 0 * x over the eight 16-bit elements of v and `sum`: NaN where one of them is not finite.
__device__ __forceinline__ __half2 zero_times(uint4 v, __half2 sum) {
    const __half2* x = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int u = 0; u < 4; ++u) sum = __hfma2(x[u], __half2half2(__ushort_as_half(0)), sum);
    return sum;
}
__device__ __forceinline__ __nv_bfloat162 zero_times(uint4 v, __nv_bfloat162 sum) {
    const __nv_bfloat162* x = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int u = 0; u < 4; ++u) sum = __hfma2(x[u], __bfloat162bfloat162(__ushort_as_bfloat16(0)), sum);
    return sum;
}

// Rows [lo, hi) of a tile without infinities and NaN, by a whole warp; true: there were any.
template <class T, int NP, int KT> __device__ __forceinline__ bool make_rows_finite(uint32_t tile, int lo, int hi) {
    using Two = typename std::conditional<Elem<T>::dtype == DVATTN_BFLOAT16, __nv_bfloat162, __half2>::type;
    bool odd = false;
#pragma unroll 1
    for (int i = (int)(threadIdx.x & 31); i < KT * NP; i += 32) {  // a panel of a row
        const int y = i / KT, r = i % KT;
        if (r < lo || r >= hi) continue;
        const uint32_t at = tile + (uint32_t)(y * KT * 128 + r * 128);
        uint4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)  // 8 neighbouring rows' chunks c ^ (r & 7) lie in different banks
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v[c].x), "=r"(v[c].y), "=r"(v[c].z), "=r"(v[c].w)
                         : "r"(at + (uint32_t)((c ^ (r & 7)) << 4))
                         : "memory");
        uint32_t zero = 0u;
        Two sum[2] = {*reinterpret_cast<Two*>(&zero), *reinterpret_cast<Two*>(&zero)};
#pragma unroll
        for (int c = 0; c < 8; ++c) sum[c & 1] = zero_times(v[c], sum[c & 1]);
        const Two all = __hadd2(sum[0], sum[1]);
        if (!__hbeq2(all, all)) {
            odd = true;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                const uint32_t a = at + (uint32_t)(c << 4);
                uint4 x;
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(a) : "memory");
                if (make_finite<T>(x))
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
            }
        }
    }
    return __any_sync(0xffffffffu, odd);
}

// `take_run(n, run)`, `wait(barrier, phase)`: as a whole warp, false when they give up.
// `opened(run)` is called at the beginning of a run, after its first window has been requested
// where that is this warp's.  `at`: {} at first.  false: a wait gave up; everything that was requested has landed.
// PARTS: a window comes as that many tiles of E / PARTS columns, one after the other, each in a
// stage of its own.
//
// The ring belongs to this warp and one consumer, so both see every phase of its barriers: a
// parity cannot be taken for the one two phases before.
//
// A warp takes about 75 cycles to issue a box.  With pages of 16 keys that is 1200 cycles for a
// window of 128 keys of one tensor, as long as HBM takes to bring it; hence `of`.
template <class T, int E, int KT, int PARTS, class Finite, class Take, class Wait, class Stop, class Opened>
__device__ __forceinline__ bool produce_windows(Producer& at, const TurnSplit& p, const WindowSource& s, const Finite& fin, int stages, uint32_t ring, uint32_t full,
                                                uint32_t empty, Take take_run, Wait wait, Stop stopped, Opened opened) {
    static_assert(Finite::always || PARTS == 1, "a tile is a window");
    constexpr int NP = E / 64 / PARTS, KPANEL = KT * 128, KTILE = NP * KPANEL;  // of a part
    const int lane = threadIdx.x & 31;
    const int h = s.h, Hkv = s.Hkv;
    // what the kernel before wrote with ordinary stores is read by TMA
    asm volatile("fence.proxy.async;" ::: "memory");
    SplitRun& run = at.run;
    int &nr = at.nr, &x = at.x, &iw = at.iw;
    bool &fresh = at.fresh, ok = true;
    // the next run; one that is left to a call for another kind of tiles looks like the end
    auto take = [&] {
        if (!take_run(nr++, run)) return false;
        if constexpr (Finite::always)
            if (fin.leave && (run.how & RUN_MIXED)) at.left = run.n, run.n = 0;
        return true;
    };
    if (nr == 0) {
        x = s.me, iw = 0, fresh = true;
        ok = take();
    } else {
        run.n = at.left;
    }
    auto finite = [&](int tile, int lo, int hi) {
        if (make_rows_finite<T, NP, KT>(ring + (uint32_t)(tile % stages * KTILE), lo, hi) && lane == 0) fin.found(run);
        fence_proxy_async_smem();
        __syncwarp();
    };
    // after a window (or none) of this warp: opens the run, goes on to the next window
    auto advance = [&](bool requested) {
        if (fresh && run.n) {
            fresh = false;
            if (!opened(run)) return false;
        }
        if (requested) x += s.of;
        while (run.n && x >= run.n) {
            x = s.me;
            if (!take()) return false;
            if (run.n && x >= run.n) {  // a run without a window of this warp
                if (!opened(run)) return false;
                continue;
            }
            fresh = true;
        }
        return true;
    };
    if (ok && run.n && x >= run.n) ok = advance(false);
    if (s.box) {
        if (lane == 0) {
            prefetch_tmap(s.map);
            if (s.tail) prefetch_tmap(s.tail_map);
        }
        const int boxes = KT / s.box, absent = -2 * p.BS;  // a coordinate that loads zeros
        int next = 0;  // first token of the lane's box of the window to be requested
        uint32_t raw_phases = 0;  // parity of each stage's `raw`
        auto find = [&] {
            const int k0 = run.k0 + x * KT;
            next = absent;
            if (run.f == p.F) {
                next = (run.w * Hkv + h) * p.tail + k0;
            } else if (lane < boxes) {
                const int l = k0 + lane * s.box, pos = run.off + l;
                if (l + s.box > 0 && l < run.sp) {
                    const int page = __ldg(p.bt + (size_t)run.w * p.maxb + pos / p.BS);
                    if (page >= 0 && page < p.NB) next = page * p.BS + pos % p.BS;
                }
            }
        };
        // The windows of a mixed run: the one before is looked through while this one lands.
        auto mixed_run = [&] {
            int held = -1, lo = 0, hi = 0;  // a tile to be looked through, its seen rows
            auto settle = [&] {
                if (held < 0) return true;
                const int st = held % stages;
                if (!wait(fin.raw + 8 * st, raw_phases >> st)) return false;
                raw_phases ^= 1u << st;
                finite(held, lo, hi);
                if (lane == 0) mbar_arrive(full + 8 * st);
                held = -1;
                return true;
            };
            bool ok = true;
            for (bool last = false; ok && !last; ++iw) {
                const int st = iw % stages, k0 = run.k0 + x * KT, n = min(KT, run.sp - k0);
                if (iw >= stages) {
                    if (!__all_sync(0xffffffffu, mbar_try_wait(empty + 8 * st, (iw / stages - 1) & 1)) && !(ok = settle())) break;
                    if (stopped() || !(ok = wait(empty + 8 * st, iw / stages - 1))) {
                        ok = false;
                        break;
                    }
                }
                const bool look = fin.look(run, k0 + n);
                const uint32_t landed = look ? fin.raw + 8 * st : full + 8 * st;
                const int z = next;
                if (lane == 0) mbar_expect_tx(landed, (uint32_t)KTILE);
                __syncwarp();
                if (lane < boxes)
#pragma unroll
                    for (int y = 0; y < NP; ++y)
                        tma_load_3d_hint(ring + (uint32_t)(st * KTILE + y * KPANEL + lane * s.box * 128), s.map, y * 64, h, z, landed, s.policy);
                if (!(ok = settle())) {  // what has just been requested lands before this returns
                    mbar_wait(landed, (look ? raw_phases >> st : iw / stages) & 1);
                    break;
                }
                if (look) held = iw, lo = max(-k0, 0), hi = n;
                last = fresh || x + s.of >= run.n;  // advance() may wait, or leave the run
                if (last) {
                    if (!(ok = settle())) break;
                } else {
                    x += s.of;
                    find();
                }
            }
            if (held >= 0) mbar_wait(fin.raw + 8 * (held % stages), raw_phases >> (held % stages) & 1);  // a wait gave up
            return ok;
        };
        if (ok && run.n) find();
        while (ok && run.n) {
            if constexpr (!Finite::always)
                if (fin.in(run)) {
                    if (!(ok = mixed_run()) || !(ok = advance(true))) break;
                    if (run.n) find();
                    continue;
                }
            const int z = next;
            const bool tail = run.f == p.F;
            for (int part = 0; part < PARTS; ++part, ++iw) {
                const int st = iw % stages;
                if (iw >= stages && (stopped() || !wait(empty + 8 * st, iw / stages - 1))) {
                    ok = false;
                    break;
                }
                if (iw == s.stall) continue;
                if (lane == 0) mbar_expect_tx(full + 8 * st, (uint32_t)KTILE);
                __syncwarp();
                const uint32_t dst = ring + (uint32_t)(st * KTILE);
                if (tail ? lane == 0 : lane < boxes)
#pragma unroll
                    for (int y = 0; y < NP; ++y)
                        tma_load_3d_hint(dst + (uint32_t)(y * KPANEL + lane * s.box * 128), tail ? s.tail_map : s.map, (part * NP + y) * 64,
                                         tail ? 0 : h, z, full + 8 * st, s.policy);
            }
            if (!ok || !(ok = advance(true))) break;
            if (run.n) find();
        }
        if (!ok)  // bounded waits
            for (int y = max(0, iw - stages); y < iw; ++y)
                if (y != s.stall) mbar_wait(full + 8 * (y % stages), (y / stages) & 1);
        return ok;
    }
    const T* cache = static_cast<const T*>(s.cache);
    const T* draft = static_cast<const T*>(s.tail);
    constexpr int NR = KT / 32;          // rows of a window whose addresses a lane finds
    constexpr int CH = E / 8 / PARTS;    // 16-byte chunks of a row of a part
    constexpr int RPI = 32 / CH;         // rows per copy instruction
    const T* next[NR];                   // rows lane + 32 k of the window to be requested, null: zeros
    auto find = [&] {
        const int k0 = run.k0 + x * KT;
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int l = k0 + lane + 32 * k;
            next[k] = nullptr;
            if (l >= run.sp) continue;
            if (run.f == p.F) {
                if (__ldcg(s.anc + ((size_t)run.w * p.tail + l) * s.SW + (l >> 5)) >> (l & 31) & 1u)
                    next[k] = draft + (((size_t)run.w * Hkv + h) * p.tail + l) * E;
            } else {
                const int pos = run.off + l;
                const int page = __ldg(p.bt + (size_t)run.w * p.maxb + pos / p.BS);
                if (page >= 0 && page < p.NB) next[k] = cache + (((size_t)page * p.BS + pos % p.BS) * Hkv + h) * E;
            }
        }
    };
    int signalled = iw;               // tiles handed over
    auto hand_over = [&](int upto) {  // their copies have landed
        fence_proxy_async_smem();
        for (; signalled < upto; ++signalled)
            if (signalled != s.stall) mbar_arrive(full + 8 * (signalled % stages));
    };
    if (ok && run.n) find();
    while (ok && run.n) {
        for (int part = 0; part < PARTS; ++part, ++iw) {
            const int st = iw % stages;
            if (iw >= stages && !__all_sync(0xffffffffu, mbar_try_wait(empty + 8 * st, (iw / stages - 1) & 1))) {
                // about to wait: hand over what is under way first
                cp_async_wait<0>();
                hand_over(iw);
                if (stopped() || !wait(empty + 8 * st, iw / stages - 1)) {
                    ok = false;
                    break;
                }
            }
            const uint32_t dst = ring + (uint32_t)(st * KTILE);
            const int ch = lane % CH;
#pragma unroll
            for (int k = 0; k < NR; ++k) {
                const unsigned long long row = reinterpret_cast<unsigned long long>(next[k]);
#pragma unroll 4
                for (int y = 0; y < CH; ++y) {
                    const int rl = y * RPI + lane / CH, r = 32 * k + rl;
                    const T* src = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, row, rl));
                    cp_async16_zfill(dst + (uint32_t)((ch >> 3) * KPANEL + r * 128 + (((ch & 7) ^ (r & 7)) << 4)),
                                     src ? src + (part * CH + ch) * 8 : cache, src ? 16 : 0);
                }
            }
            cp_async_commit();
            if constexpr (!Finite::always)
                if (fin.in(run)) {
                    const int k0 = run.k0 + x * KT, n = min(KT, run.sp - k0);
                    if (fin.look(run, k0 + n)) {
                        cp_async_wait<0>();
                        __syncwarp();
                        hand_over(iw);
                        finite(iw, max(-k0, 0), n);
                        hand_over(iw + 1);
                        continue;
                    }
                }
            cp_async_wait<1>();
            hand_over(iw);
        }
        if (!ok) break;
        if (fresh || x + s.of >= run.n) {  // advance() may wait
            cp_async_wait<0>();
            hand_over(iw);
        }
        if (!(ok = advance(true))) break;
        if (run.n) find();
    }
    cp_async_wait<0>();
    if (ok) hand_over(iw);
    return ok;
}

}  // namespace dvb
