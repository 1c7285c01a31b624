// Draft-tree attention on the 5th-generation tensor cores (tcgen05 + TMEM), 16-bit types.
//
// A CTA walks a range of key windows (turns.cuh).  Jobs: a job is S = Q K^T of one 128-row
// query tile and one window, its softmax, and O += P V.  Job j uses score buffer j & 1 of
// TMEM, and the tensor core issues S(j + 1) before PV(j), so it works for one job while the
// other's softmax runs.  Two forms, by the rows S * G of a KV head:
//   more than 128 rows (head dims 64, 128): bound by the softmax-PV-S chain.  Two row tiles
//     share every 128-key window; j & 1 is the tile, each with its own softmax warpgroup.
//   up to 128 rows, and head dim 256: bound by HBM.  One tile, 64-key windows, one softmax
//     warpgroup, half an SM (head dim 256: a whole one): what the beginning and end of a
//     piece cost one CTA is hidden behind the other's stream.
// Warps: 4 per softmax group (a thread owns one query row = one TMEM lane), one that walks the
// range (split_schedule), one MMA issuer, one K (and Q) and one V producer.  Producers fill
// swizzled rings with TMA boxes where pages and windows are whole numbers of boxes of 8 or more
// rows (page sizes that are multiples of 8), else they gather rows with cp.async.  What lies in
// rows that nobody sees never matters: their scores are masked, and their V rows are zeroed
// before PV (0 * NaN is NaN).  An infinity or NaN of a value that some tokens see and others do not is
// a zero for PV, too, and tree_merge_kernel adds it to who sees it: drafted values come from the prep
// kernel's copy, and the V producer looks through the windows in which the tokens' locations differ (a call
// in which they differ everywhere takes 1.3 to 1.5 times as long; one in which they do not, 1 to 2%).
//
// Measured with prep and merge: 32 sequences of two turns, 64/4 heads, 8 tokens, 337 MB: 88 to 92 us
// by the box, 57 to 59% of HBM's copy rate (203 with one CTA per SM, rows gathered and rotated by its own threads); the
// stream alone reaches 89% with 128 rows, 98% with 32.  4 sequences of up to 131072 keys, 128/8
// heads, 16 tokens (two tiles): 557 to 590 us, 688 to 650 TFLOP/s, 4325 cycles per 128-key window at
// the 1.5 GHz that the power limit leaves; tensor core and SFU are each busy for a third of the time.
//
// Every wait is bounded; one that gives up sets the call's error word, ends the CTA with
// nothing in flight, and tree_merge_kernel writes NaN to all outputs of the call.
#include "tcgen05.cuh"
#include "tma_host.cuh"
#include "tree.cuh"
#include "windows.cuh"

namespace dvb {

template <int E, bool TWO> struct TcCfg {
    static constexpr int KT = TWO ? 128 : 64;       // keys per window
    static constexpr int NG = TWO ? 2 : 1;          // row tiles, softmax warpgroups, O accumulators
    static constexpr int CTAS = TWO || E == 256 ? 1 : 2;  // per SM
    static constexpr int NP = E / 64;               // 64-column panels
    static constexpr int QPANEL = 128 * 128, KPANEL = KT * 128, QTILE = NP * QPANEL, KTILE = NP * KPANEL;
    static constexpr int NT = (4 * NG + 4) * 32;    // the last warpgroup: MMA, K, V, the walk
    static constexpr int WARP_MMA = 4 * NG, WARP_K = 4 * NG + 1, WARP_V = 4 * NG + 2, WARP_WALK = 4 * NG + 3;
    // Registers of a softmax thread and of the others, out of an even share of 168 (two tiles,
    // 384 threads) or 128 (256 threads, two CTAs): 256 * 208 + 128 * 88 = 384 * 168 and
    // 128 * 168 + 128 * 88 = 256 * 128.  A row of 64 scores fits in 168 (the batched decode took half as
    // long again with 128 of them, which spilled); with 128 scores 208 still spill 108 bytes a thread.
    // 0: every thread may have 255.
    static constexpr int REGS = TWO ? 208 : E == 256 ? 0 : 168;
    // Shared memory: sets of Q tiles (a second one lets the next turn's or piece's arrive while
    // the last one is in use), the K ring, the V ring.
    static constexpr int Q_SETS = E == 64 ? 2 : 1, K_STAGES = E == 64 ? 4 : E == 256 ? 2 : 3, VS = E == 64 ? 4 : E == 256 ? 3 : 2;
    static constexpr int Q_SET = NG * QTILE;
    static constexpr int OFF_K = Q_SETS * Q_SET, OFF_V = OFF_K + K_STAGES * KTILE, OFF_BAR = OFF_V + VS * KTILE;
    static constexpr int OFF_MISC = OFF_BAR + 48 * 8;
    static constexpr int OFF_RUN = OFF_MISC + 32;
    static constexpr int SMEM = OFF_RUN + RUN_RING * (int)sizeof(SplitRun);
    static_assert(SMEM <= (CTAS == 2 ? 115712 : 232448), "more shared memory than a CTA may use");
    // The softmax warps wait for v_full and v_empty in some phases only.  They cannot take the phase before
    // for the one they wait for: a job's S is complete after the PV of two jobs before, which used V's
    // stage for the last time before this window if the stages are two or more.
    static_assert(VS >= 2, "a phase of v_full or v_empty could be taken for another");
    // TMEM columns: scores (P over them) at 0 and KT, O
    static constexpr int COLS = CTAS == 2 ? 256 : 512, TM_O = CTAS == 2 ? 128 : 256;
};

// How far (log2) the softmax's reference point lies below the maximum it was taken from.  fp16 is
// normal down to 2^-14 and zero below 2^-25: weights relative to the maximum itself lose their bits
// 10 nats under it and are gone at 17, where a long context still has thousands of keys, while the
// sum counts them.  With the maximum 8 above the reference at most, 2^15 is the largest weight, and a
// weight is rounded by half an ulp or by 2^-32 of the row's largest one, whichever is more.
template <class T> constexpr float kRefBelow = 0.f;  // bf16 has the range of the sums
template <> constexpr float kRefBelow<__half> = 7.f;

// 32 bytes in one store (the address a multiple of 32).
__device__ __forceinline__ void store_sector(void* dst, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

__device__ __forceinline__ void mark_odd(const TreeParams& p, int wh) {  // tells the merge
    p.odd_any[wh] = 1;
    p.header[2] = 1;
}

// The V producer's part in values that are not finite (windows.cuh).
struct OddValues {
    static constexpr bool always = false;
    const TreeParams& p;
    int h;
    uint32_t raw;
    __device__ __forceinline__ bool in(const SplitRun& run) const { return run.how & RUN_MIXED; }
    __device__ __forceinline__ bool look(const SplitRun& run, int end) const { return __ldcg(p.same + (size_t)run.w * p.F + run.f) < end; }
    __device__ __forceinline__ void found(const SplitRun& run) const { mark_odd(p, run.w * p.Hkv + h); }
};

template <class T, int E, bool TWO>
__global__ void __launch_bounds__(TcCfg<E, TWO>::NT, TcCfg<E, TWO>::CTAS) tree_tc_kernel(TreeParams p, const __grid_constant__ TreeMaps maps) {
    using C = TcCfg<E, TWO>;
    constexpr int KT = C::KT, NG = C::NG, VS = C::VS;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t s0 = smem_u32(smem);
    if (s0 & 1023) {  // the swizzle's period
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (tid == 0) atomicOr(p.header + 3, 4);
        return;
    }
    const bool bf16 = Elem<T>::dtype == DVATTN_BFLOAT16;
    const uint32_t bar = s0 + C::OFF_BAR;
    const uint32_t k_full = bar, k_empty = bar + 32, v_full = bar + 64, v_empty = bar + 96;
    const uint32_t s_full = bar + 128, p_full = bar + 144, q_full = bar + 160, q_empty = bar + 176, o_done = bar + 192;
    const uint32_t run_full = bar + 200, run_empty = run_full + 8 * RUN_RING, v_raw = run_empty + 8 * RUN_RING;  // 45 in all
    SplitRun* runs = reinterpret_cast<SplitRun*>(smem + C::OFF_RUN);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 8);
    if (tid == 0) {
        for (int s = 0; s < 4; ++s) {
            mbar_init(k_full + 8 * s, p.box ? 1 : 32);
            mbar_init(k_empty + 8 * s, 1);
            mbar_init(v_full + 8 * s, p.box ? 1 : 32);
            mbar_init(v_empty + 8 * s, 1);
            mbar_init(v_raw + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(s_full + 8 * s, 1);
            mbar_init(p_full + 8 * s, 128);
            mbar_init(q_full + 8 * s, 1);
            mbar_init(q_empty + 8 * s, 1);
        }
        for (int s = 0; s < RUN_RING; ++s) {
            mbar_init(run_full + 8 * s, 1);
            mbar_init(run_empty + 8 * s, 3 + 4 * NG);  // MMA, K, V, the softmax warps
        }
        mbar_init(o_done, 1);
        *s_abort = 0;
        fence_mbar_init();
    }
    if (wid == C::WARP_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s0 + C::OFF_MISC), "n"(C::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + C::OFF_MISC);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // the merge may be launched now: it reads the prep kernel's results without waiting
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    const int g = blockIdx.x / p.Hkv, h = blockIdx.x - g * p.Hkv;
    // a whole warp waits, and gives up as a whole
    auto wait = [&](uint32_t b, int phase) { return __all_sync(0xffffffffu, mbar_wait(b, phase & 1)); };
    auto wait_lazy = [&](uint32_t b, int phase) { return __all_sync(0xffffffffu, mbar_wait_lazy(b, phase & 1)); };
    auto take_run = [&](int n, SplitRun& run) {  // the n-th run, by a whole warp
        if (!wait(run_full + 8 * (n % RUN_RING), n / RUN_RING)) return false;
        run = runs[n % RUN_RING];
        __syncwarp();
        if (lane == 0) mbar_arrive(run_empty + 8 * (n % RUN_RING));
        return true;
    };
    auto give_up = [&](int bit) {
        if (lane == 0) {
            *s_abort = 1;
            atomicOr(p.header + 3, bit);
        }
    };

    // A piece's query tiles, again for each turn (the drafted keys keep the last turn's); by the
    // K producer.  false: a wait gave up, nothing was requested.
    auto load_q = [&](const SplitRun& run, int epoch) {
        const int set = epoch % C::Q_SETS;
        if (epoch >= C::Q_SETS && (*s_abort || !wait(q_empty + 8 * set, epoch / C::Q_SETS - 1))) return false;
        if (lane == 0) {
            mbar_expect_tx(q_full + 8 * set, (uint32_t)C::Q_SET);
            const int z = ((min(run.f, p.F - 1) * p.W + run.w) * p.Hkv + h) * p.rows + run.t * p.mi;
            for (int t = 0; t < NG; ++t)
#pragma unroll
                for (int x = 0; x < C::NP; ++x)
                    tma_load_3d(s0 + (uint32_t)(set * C::Q_SET + t * C::QTILE + x * C::QPANEL), &maps.q, x * 64, 0, z + 128 * t, q_full + 8 * set);
        }
        __syncwarp();
        return true;
    };
    if (wid >= C::WARP_MMA) {
        if constexpr (C::REGS > 0) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (wid == C::WARP_K || wid == C::WARP_V) {
        const bool is_k = wid == C::WARP_K;
        WindowSource src;
        src.cache = is_k ? p.k : p.v, src.tail = is_k ? p.dkr : p.dvr;
        src.map = is_k ? &maps.k : &maps.v, src.tail_map = is_k ? &maps.dk : &maps.dv;
        src.h = h, src.Hkv = p.Hkv, src.box = p.box, src.me = 0, src.of = 1, src.anc = p.anc, src.SW = p.SW;
        // keys and values that one row tile reads are read once: they leave L2 first, the partial
        // results stay for the merge
        src.policy = p.nt == 1 ? l2_evict_first() : l2_evict_normal();
        src.stall = is_k && blockIdx.x == 0 ? p.stall_tile : -1;
        int epoch = 0;
        Producer at{};
        auto stopped = [&] { return *s_abort != 0; };
        auto opened = [&](const SplitRun& run) { return !is_k || !(run.how & RUN_Q_NEW) || load_q(run, epoch++); };
        bool ok = produce_windows<T, E, KT, 1>(at, p, src, AsTheyAre{!is_k}, is_k ? C::K_STAGES : VS, s0 + (is_k ? C::OFF_K : C::OFF_V),
                                               is_k ? k_full : v_full, is_k ? k_empty : v_empty, take_run, wait, stopped, opened);
        // values from the first mixed run on: code of its own, which would cost every window 5% in the loop before
        if (ok && at.left)
            ok = produce_windows<T, E, KT, 1>(at, p, src, OddValues{p, h, v_raw}, VS, s0 + C::OFF_V, v_full, v_empty, take_run, wait, stopped,
                                              [](const SplitRun&) { return true; });
        if (!ok) {
            give_up(1);
            if (is_k)  // what load_q requested lands before the CTA can exit, too
                for (int y = max(0, epoch - C::Q_SETS); y < epoch; ++y) mbar_wait(q_full + 8 * (y % C::Q_SETS), (y / C::Q_SETS) & 1);
        }
    } else if (wid == C::WARP_WALK) {
        auto tail = [&](int w) {  // are there odd drafted values?
            const int wh = w * p.Hkv + h;
            for (int s = lane; s < p.S; s += 32)
                if (__ldcg(p.odd + (size_t)wh * p.S + s)) mark_odd(p, wh);
            __syncwarp();
        };
        if (!split_schedule(p, lane, g, runs, run_full, run_empty, [&] { return *s_abort != 0; }, 1, tail)) give_up(1);
    } else if (wid == C::WARP_MMA) {
        // =================================== MMA ===================================
        // (the whole warp converged: umma_warp)
        const uint32_t id_s = idesc(bf16, 128, KT, false), id_o = idesc(bf16, 128, E, true);
        const uint64_t dq0 = sdesc(s0, 16, 1024), dk0 = sdesc(s0 + C::OFF_K, 16, 1024), dv0 = sdesc(s0 + C::OFF_V, C::KPANEL, 1024);
        {
            int j = 0, ks = 0, kp = 0, vs = 0, vp = 0, qs = 0, qp = 0, piece = 0;
            bool ok = true;
            // PV of job jj, the n-th of its piece, over the V window at hand; `last`: its last use
            auto issue_pv = [&](int jj, int n, bool last) {
                const int b = jj & 1;
                if (!wait(v_full + 8 * vs, vp) || !wait(p_full + 8 * b, jj >> 1)) return false;
                tc_fence_after();
                const uint64_t b0 = dv0 + (uint64_t)((vs * C::KTILE) >> 4);
                const uint32_t d = tmem + C::TM_O + (TWO ? 128 * b : 0), a = tmem + KT * b;
                const uint32_t acc = n >= NG;  // the first PV of an O in a piece overwrites it
#pragma unroll
                for (int kk = 0; kk < KT / 16; ++kk) umma_ts_warp(d, a + 8 * kk, b0 + (uint64_t)((kk * 16 * 128) >> 4), id_o, kk > 0 ? 1u : acc);
                if (last) {
                    umma_commit_warp(v_empty + 8 * vs);
                    if (++vs == VS) vs = 0, vp ^= 1;
                }
                return true;
            };
            SplitRun run;
            int nr = 0, n = 0;  // runs taken, jobs of the piece issued
            while ((ok = take_run(nr++, run)) && run.n) {
                if (run.how & RUN_FIRST) n = 0;
                if ((run.how & RUN_Q_NEW) && !(ok = wait(q_full + 8 * qs, qp))) break;
                const uint64_t qd = dq0 + (uint64_t)((qs * C::Q_SET) >> 4);
                for (int x = 0; ok && x < run.n; ++x) {
                    if (!(ok = wait(k_full + 8 * ks, kp))) break;
                    for (int t = 0; ok && t < NG; ++t, ++j, ++n) {
                        tc_fence_after();
                        const uint64_t a0 = qd + (uint64_t)((t * C::QTILE) >> 4), b0 = dk0 + (uint64_t)((ks * C::KTILE) >> 4);
#pragma unroll
                        for (int kk = 0; kk < E / 16; ++kk)
                            umma_warp(tmem + KT * (j & 1), a0 + (uint64_t)(((kk >> 2) * C::QPANEL + (kk & 3) * 32) >> 4),
                                 b0 + (uint64_t)(((kk >> 2) * C::KPANEL + (kk & 3) * 32) >> 4), id_s, kk > 0 ? 1u : 0u);
                        umma_commit_warp(s_full + 8 * (j & 1));
                        if (t == NG - 1) {
                            umma_commit_warp(k_empty + 8 * ks);
                            if ((run.how & RUN_Q_END) && x + 1 == run.n) umma_commit_warp(q_empty + 8 * qs);
                        }
                        if (n > 0) ok = issue_pv(j - 1, n - 1, !TWO || t == 0);
                    }
                    if (++ks == C::K_STAGES) ks = 0, kp ^= 1;
                }
                if (!ok) break;
                if ((run.how & RUN_Q_END) && ++qs == C::Q_SETS) qs = 0, qp ^= 1;
                if (run.how & RUN_LAST) {
                    if (!(ok = issue_pv(j - 1, n - 1, true))) break;
                    umma_commit_warp(o_done);
                    ++piece;
                }
            }
            if (!ok) {
                give_up(2);
                // all issued MMAs have completed before TMEM is released
                umma_commit_warp(o_done);
                mbar_wait(o_done, piece & 1);
            }
        }
    }
    } else {
        // ================================= softmax =================================
        if constexpr (C::REGS > 0) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS));
        const int grp = wid >> 2, r = (wid & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((wid & 3) * 32) << 16;
        const uint32_t tO = tmem + lanes + C::TM_O + 128 * grp;
        int j = 0, iw = 0, piece = 0;
        int tok = 0, orow = 0;          // this thread's row of the piece at hand: token, output row
        bool in = false, live = false;  // it is one; the warp has one
        // One run after the other; a finished piece's result is written once the next run's limit
        // is on its way.
        float m = neg_inf(), l = 0.f;  // running maximum (log2 units, stepped) and sum
        int mine = 0, nr = 0, was_row = 0;  // jobs of the piece done, runs taken
        bool pending = false, whole = false, was_in = false, was_live = false;
        size_t prow = 0;
        SplitRun run;
        bool ok;
        while ((ok = take_run(nr++, run))) {
            if (run.how & RUN_FIRST) {
                const int row = run.t * p.mi + grp * 128 + r;
                in = row < p.rows;
                tok = in ? row / p.G : 0;
                orow = (run.w * p.Hq + h * p.G + (in ? row - tok * p.G : 0)) * p.S + tok;
                live = __any_sync(0xffffffffu, in);
            }
            const bool tail = run.f == p.F;
            int lim = 0;  // keys of the turn that the row sees
            if (run.n && in && !tail) lim = __ldcg(p.lim + ((size_t)run.f * p.W + run.w) * p.S + tok);
            if (pending) {
                // ---- the piece's result ----
                if (!(ok = wait(o_done, piece))) break;
                tc_fence_after();
                const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
                const float lse2 = l == 0.f ? neg_inf() : m + log2f(l);
#pragma unroll 1
                for (int c = 0; c < E / 32; ++c) {
                    float ov[32];
                    if (was_live) {
                        tmem_ld32(tO + 32 * c, ov);
                        tmem_wait_ld();
                        reg_fence<32>(ov);
#pragma unroll
                        for (int u = 0; u < 32; ++u) ov[u] *= inv;
                    }
                    if (l == 0.f)  // a token that is not there, a piece without a key that it sees
#pragma unroll
                        for (int u = 0; u < 32; ++u) ov[u] = 0.f;
                    if (was_in) {
                        // a thread writes whole 32-byte sectors of its row
                        uint32_t x[32];
                        if (whole) {
                            T* op = static_cast<T*>(p.out) + (size_t)was_row * E + 32 * c;
#pragma unroll
                            for (int u = 0; u < 16; ++u) x[u] = Elem<T>::pack2(ov[2 * u], ov[2 * u + 1]);
                            if (p.out_sectors) {
#pragma unroll
                                for (int u = 0; u < 2; ++u) store_sector(op + 16 * u, x + 8 * u);
                            } else {
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    *reinterpret_cast<uint4*>(op + 8 * u) = make_uint4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
                            }
                        } else {
#pragma unroll
                            for (int u = 0; u < 32; ++u) x[u] = __float_as_uint(ov[u]);
#pragma unroll
                            for (int u = 0; u < 4; ++u) store_sector(p.part_o + prow * E + 32 * c + 8 * u, x + 8 * u);
                        }
                    }
                }
                if (was_in) {
                    if (!whole) p.part_lse[prow] = lse2;
                    else if (p.lse_out) p.lse_out[was_row] = lse2 * kLn2;
                }
                pending = false;
                ++piece;
                m = neg_inf(), l = 0.f;
                mine = 0;
            }
            if (!run.n) break;
            // ---- this group's jobs of the run's windows ----
            for (int x0 = 0; x0 < run.n; ++x0) {
                const int job = j + NG * x0 + grp, b = job & 1;
                const int k0 = run.k0 + x0 * KT, n = min(KT, run.sp - k0);
                const uint32_t tS = tmem + lanes + KT * b;
                // drafted keys: the row's ancestors among them, and whether the thread's V row counts
                uint32_t anc[KT / 32];
                bool v_seen = r < n && k0 + r >= 0;
                if (tail) {
                    const uint32_t* words = p.anc + (size_t)run.w * p.S * p.SW;
                    const int key = k0 + r;
#pragma unroll
                    for (int x = 0; x < KT / 32; ++x) anc[x] = in ? __ldcg(words + (size_t)tok * p.SW + (k0 >> 5) + x) : 0u;
                    if (v_seen) v_seen = __ldcg(words + (size_t)key * p.SW + (key >> 5)) >> (key & 31) & 1u;
                }
                if (!wait(s_full + 8 * b, job >> 1)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (live) {
                    float sv[KT];
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c) tmem_ld32(tS + 32 * c, *reinterpret_cast<float(*)[32]>(sv + 32 * c));
                    tmem_wait_ld();
                    reg_fence<KT>(sv);
                    // the maximum is taken before scaling and masked scores are -inf: a scale that is
                    // not positive goes into the scores first
                    const float sl2 = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
                    if (p.scale_log2 <= 0.f)
#pragma unroll
                        for (int c = 0; c < KT; ++c) sv[c] = p.scale_log2 == 0.f ? 0.f : -sv[c];
                    if (tail || !__all_sync(0xffffffffu, k0 >= 0 && lim - k0 >= KT)) {
#pragma unroll
                        for (int x = 0; x < KT / 32; ++x) {
                            uint32_t see;
                            if (tail) {
                                see = anc[x];
                            } else {
                                const int d = lim - k0 - 32 * x, e = -k0 - 32 * x;  // columns in front of d, not of e
                                see = d >= 32 ? 0xffffffffu : d <= 0 ? 0u : (1u << d) - 1;
                                see &= e <= 0 ? 0xffffffffu : e >= 32 ? 0u : 0xffffffffu << e;
                            }
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (!(see >> c & 1u)) sv[32 * x + c] = neg_inf();
                        }
                    }
                    float mx[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) mx[u] = sv[u];
#pragma unroll
                    for (int c = 8; c < KT; c += 16)
#pragma unroll
                        for (int u = 0; u < 8; ++u) mx[u] = fmax3(mx[u], sv[c + u], sv[c + 8 + u < KT ? c + 8 + u : c + u]);
                    const float mxs = fmax3(fmax3(mx[0], mx[1], mx[2]), fmax3(mx[3], mx[4], mx[5]), fmaxf(mx[6], mx[7])) * sl2 - kRefBelow<T>;
                    // the reference point moves only when the maximum grows by more than 8 (a
                    // factor 256 in the exponentials); the result is exact either way
                    const float mnew = mxs > m + 8.f ? mxs : m;
                    const float alpha = mnew == m ? 1.f : ex2(m - mnew);
                    const float mu = mnew == neg_inf() ? 0.f : mnew;
                    const uint64_t sc2 = f2u(sl2, sl2), nmu2 = f2u(-mu, -mu);
                    uint64_t ps2[4] = {0ull, 0ull, 0ull, 0ull};
                    // P is rounded to T, the tensor core's operand next to V (half an ulp of T a
                    // weight, and see kRefBelow); the sum is of the unrounded weights
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c) {
                        uint32_t pk[16];
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            float x0, x1;
                            u2f(ffma2(f2u(sv[32 * c + 2 * u], sv[32 * c + 2 * u + 1]), sc2, nmu2), x0, x1);
                            const float e0 = ex2(x0), e1 = ex2(x1);
                            ps2[u & 3] = fadd2(ps2[u & 3], f2u(e0, e1));
                            pk[u] = Elem<T>::pack2(e0, e1);
                        }
                        tmem_st16(tS + 16 * c, pk);
                    }
                    float a0, a1;
                    u2f(fadd2(fadd2(ps2[0], ps2[1]), fadd2(ps2[2], ps2[3])), a0, a1);
                    l = l * alpha + (a0 + a1);
                    m = mnew;
                    if (mine > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        // O holds the PV of this tile's earlier jobs.  With two tiles they completed
                        // before this S was signalled (S(j) is issued after PV(j - 2)); with one, the
                        // last of them is PV(j - 1), whose completion frees its V window.
                        if (NG == 1 && !wait(v_empty + 8 * ((iw + x0 - 1) % VS), (iw + x0 - 1) / VS)) {
                            ok = false;
                            break;
                        }
                        if (NG == 1) tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < E / 32; ++c) {
                            float ov[32];
                            tmem_ld32(tO + 32 * c, ov);
                            tmem_wait_ld();
                            reg_fence<32>(ov);
#pragma unroll
                            for (int u = 0; u < 32; ++u) ov[u] *= alpha;
                            tmem_st32(tO + 32 * c, ov);
                        }
                    }
                    tmem_wait_st();
                }
                if (p.box && grp == 0 && (tail || k0 < 0 || n < KT)) {
                    // V rows of this window that nobody sees: P is 0 there
                    if (!wait(v_full + 8 * ((iw + x0) % VS), (iw + x0) / VS)) {
                        ok = false;
                        break;
                    }
                    if (r < KT && !v_seen) {
                        uint8_t* v = smem + C::OFF_V + ((iw + x0) % VS) * C::KTILE + r * 128;
#pragma unroll
                        for (int x = 0; x < C::NP; ++x)
#pragma unroll
                            for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(v + x * C::KPANEL + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                }
                tc_fence_before();
                mbar_arrive(p_full + 8 * b);
                ++mine;
            }
            if (!ok) break;
            j += NG * run.n;
            iw += run.n;
            if (run.how & RUN_LAST) {
                pending = true;
                whole = run.how & RUN_WHOLE, was_in = in, was_live = live, was_row = orow;
                prow = ((size_t)blockIdx.x * 2 + (run.how & RUN_BEGIN ? 1 : 0)) * p.mi + grp * 128 + r;
            }
        }
        if (!ok) give_up(8);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (wid == C::WARP_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::COLS) : "memory");
}

template <class T, int E, bool TWO> static TreeKernel tc_kernel() {
    using C = TcCfg<E, TWO>;
    // One sequence of 16384 keys, 128 rows: 30 us with at least 8 windows a group, 45 and 49 with 4
    // and 1 (the merge reads that many more partials); two tiles, 4 x 4096 keys: 43 us with at
    // least 4, 51 with 8.
    return TreeKernel{(const void*)&tree_tc_kernel<T, E, TWO>, C::NT, C::KT, 128 * C::NG, C::CTAS, TWO ? 4 : 8, (size_t)C::SMEM};
}
template <class T> static TreeKernel tc_pick(int E, int rows) {
    if (E == 256) return tc_kernel<T, 256, false>();
    if (rows > 128) return E == 64 ? tc_kernel<T, 64, true>() : tc_kernel<T, 128, true>();
    return E == 64 ? tc_kernel<T, 64, false>() : tc_kernel<T, 128, false>();
}
TreeKernel tree_tc_pick(int dtype, int E, int rows) {
    return dtype == DVATTN_FLOAT16 ? tc_pick<__half>(E, rows) : tc_pick<__nv_bfloat16>(E, rows);
}

bool tree_tc_maps(TreeParams& p, int dtype, int E, TreeMaps& m) {
    const long long tokens = p.NB * p.BS, drafts = (long long)p.W * p.Hkv * p.S;
    p.out_sectors = !(reinterpret_cast<uintptr_t>(p.out) & 31);
    if (!encode_cache_map(&m.q, p.qr, dtype, E, 1, (long long)p.F * p.W * p.Hq * p.S, 128)) return false;
    p.box = p.cap > 0 && drafts <= 0x7fffffffLL - p.kt ? window_box(p.BS, p.kt, p.NB) : 0;
    p.align = p.box ? p.box : 1;
    if (!p.box) return true;
    return encode_cache_map(&m.k, p.k, dtype, E, p.Hkv, tokens, p.box) && encode_cache_map(&m.v, p.v, dtype, E, p.Hkv, tokens, p.box) &&
           encode_cache_map(&m.dk, p.dkr, dtype, E, 1, drafts, p.kt) && encode_cache_map(&m.dv, p.dvr, dtype, E, 1, drafts, p.kt);
}

}  // namespace dvb
