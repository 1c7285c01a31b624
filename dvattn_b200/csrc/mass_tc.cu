// Accumulated attention weight on the 5th-generation tensor cores (tcgen05 + TMEM), 16-bit types.
//
// A job is S^T = K Q^T of one window of 128 keys (the TMEM lanes) and up to 128 query rows (the
// columns).  So a thread owns a key: it adds up the weights 2^(scale s - lse) of its key over all
// rows in registers and writes the key's mass once, with no reduction across threads and no
// partial results; every key's sum has a fixed order.
//
// A CTA walks a range of windows (turns.cuh), one KV head.  The windows of a run alternate between
// two groups (the same in every pass of rows, so a key's mass has one writer), each one K producer
// with a ring of its own, one MMA warp, two score buffers of 128 columns in TMEM and four warps
// that form the sums, so one group's products run under the other's exponentials.  The query tile of a (sequence,
// turn) stays in shared memory with its rows' lse and limits; where it holds fewer rows than there
// are, the CTA runs its windows again for each pass of rows.  Every wait is bounded (see
// tree_tc.cu); a call that gave up leaves the error word set, its sums unfinished.
//
// Bound: few rows, HBM: a decode step of 32 sequences, 154 MB, takes 35 us, 68% of its copy rate (88%
// with 128 sequences).  Many rows, the sums: 496 rows over 4 x 26000 keys take 176 us; the SFU,
// 16 exponentials a clock and SM, is busy for two thirds of the time, the tensor core for a
// third.  Twice the warps for the sums (177 us), a share of the exponentials as polynomials on
// the FMA pipe (an eighth 178 us, a quarter 185), and score buffers that are given back as soon as
// they are read (182) do not help; two scores' loads in flight across jobs cost registers (245).
#include <type_traits>

#include "mass.cuh"
#include "windows.cuh"

namespace dvb {

// ROWS: query rows of a pass, a tile set of 8 to 128 KB next to the groups' K rings.
template <int E, int ROWS_> struct MassCfg {
    static constexpr int KT = 128, NP = E / 64, ROWS = ROWS_;
    static constexpr int Q_SETS = ROWS > 64 || E == 256 ? 1 : 2;
    static constexpr int PARTS = E == 256 ? 2 : 1;  // a K window of head dim 256 comes in two tiles
    static constexpr int QPANEL = ROWS * 128, KPANEL = KT * 128, QTILE = NP * QPANEL, KTILE = NP / PARTS * KPANEL;
    static constexpr int K_STAGES = E == 64 ? 4 : QTILE > 65536 ? 1 : QTILE > 32768 ? 2 : 3;  // of a group
    static constexpr int ROWDATA = 2 * ROWS * 4;  // nlse, lim
    static constexpr int OFF_K = Q_SETS * QTILE, OFF_ROW = OFF_K + 2 * K_STAGES * KTILE, OFF_BAR = OFF_ROW + Q_SETS * ROWDATA;
    static constexpr int OFF_MISC = OFF_BAR + 48 * 8, OFF_RUN = OFF_MISC + 32, SMEM = OFF_RUN + RUN_RING * (int)sizeof(SplitRun);
    static constexpr int WARP_MMA = 8, WARP_K = 10, WARP_WALK = 12, NT = 13 * 32;  // warps 0..7 sums, two each of MMA and K
    static_assert(SMEM <= 232448, "more shared memory than a CTA may use");
};

template <class T, int E, int ROWS>
__global__ void __launch_bounds__(MassCfg<E, ROWS>::NT, 1) mass_tc_kernel(MassParams p, const __grid_constant__ MassMaps maps) {
    using C = MassCfg<E, ROWS>;
    constexpr int KT = C::KT, KS = E / 16 / C::PARTS;  // MMA steps of a tile
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
    const uint32_t k_full = bar, k_empty = bar + 64, d_full = bar + 128, d_empty = bar + 160, q_full = bar + 192, q_empty = bar + 208,
                   m_done = bar + 224, run_full = bar + 240, run_empty = run_full + 8 * RUN_RING;
    SplitRun* runs = reinterpret_cast<SplitRun*>(smem + C::OFF_RUN);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 8);
    if (tid == 0) {
        for (int s = 0; s < 8; ++s) {
            mbar_init(k_full + 8 * s, p.box ? 1 : 32);
            mbar_init(k_empty + 8 * s, 1);
        }
        for (int s = 0; s < 4; ++s) {  // [group][buffer]
            mbar_init(d_full + 8 * s, 1);
            mbar_init(d_empty + 8 * s, 4);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(q_full + 8 * s, 1);
            mbar_init(q_empty + 8 * s, 2 + 8);  // the MMA and the sum warps
            mbar_init(m_done + 8 * s, 1);
        }
        for (int s = 0; s < RUN_RING; ++s) {
            mbar_init(run_full + 8 * s, 1);
            mbar_init(run_empty + 8 * s, 4 + 8);  // MMA, K, the sum warps
        }
        *s_abort = 0;
        fence_mbar_init();
    }
    if (wid == C::WARP_MMA) {  // TMEM columns: [group][buffer] of 128 scores
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(s0 + C::OFF_MISC) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + C::OFF_MISC);
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int g = blockIdx.x / p.Hkv, h = blockIdx.x - g * p.Hkv;
    auto wait = [&](uint32_t b, int phase) { return __all_sync(0xffffffffu, mbar_wait(b, phase & 1)); };
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
    // rows of a run's pass, and its chunks of up to 128
    auto rows_of = [&](const SplitRun& run) { return min(C::ROWS, p.rows_pad - run.t * C::ROWS); };

    if (wid == C::WARP_K || wid == C::WARP_K + 1) {
        const int grp = wid - C::WARP_K;
        WindowSource src;
        src.cache = p.k, src.tail = nullptr, src.map = &maps.k, src.tail_map = nullptr, src.anc = nullptr, src.SW = 0;
        src.h = h, src.Hkv = p.Hkv, src.box = p.box, src.me = grp, src.of = 2;
        src.policy = p.passes == 1 ? l2_evict_first() : l2_evict_normal();
        src.stall = blockIdx.x == 0 && grp == 0 ? p.stall_tile : -1;
        int epoch = 0;
        // the queries of a run, their lse and limits
        auto load_q = [&](const SplitRun& run) {
            if (grp != 0 || !(run.how & RUN_Q_NEW)) return true;
            const int set = epoch % C::Q_SETS;
            if (epoch >= C::Q_SETS && (*s_abort || !wait(q_empty + 8 * set, epoch / C::Q_SETS - 1))) return false;
            const int n = rows_of(run), chunks = (n + 63) / 64;  // boxes of 64 rows; past the last row come others or zeros
            const size_t fwh = ((size_t)run.f * p.W + run.w) * p.Hkv + h, wh = (size_t)run.w * p.Hkv + h;
            if (lane == 0) {
                mbar_expect_tx(q_full + 8 * set, (uint32_t)(chunks * C::NP * 64 * 128 + 2 * n * 4));
                bulk_load(s0 + C::OFF_ROW + set * C::ROWDATA, p.nlse + wh * p.rows_pad + run.t * C::ROWS, n * 4, q_full + 8 * set);
                bulk_load(s0 + C::OFF_ROW + set * C::ROWDATA + C::ROWS * 4, p.lim + fwh * p.rows_pad + run.t * C::ROWS, n * 4, q_full + 8 * set);
            }
            __syncwarp();
            if (lane < chunks)
#pragma unroll
                for (int x = 0; x < C::NP; ++x)
                    tma_load_3d(s0 + (uint32_t)(set * C::QTILE + x * C::QPANEL + lane * 64 * 128), &maps.q, x * 64, 0,
                                (int)(fwh * p.rows_pad) + run.t * C::ROWS + lane * 64, q_full + 8 * set);
            ++epoch;
            return true;
        };
        Producer at{};
        if (!produce_windows<T, E, KT, C::PARTS>(at, p, src, AsTheyAre{false}, C::K_STAGES, s0 + C::OFF_K + grp * C::K_STAGES * C::KTILE, k_full + 32 * grp, k_empty + 32 * grp,
                                                 take_run, wait, [&] { return *s_abort != 0; }, load_q)) {
            give_up(1);
            for (int y = max(0, epoch - C::Q_SETS); y < epoch; ++y) mbar_wait(q_full + 8 * (y % C::Q_SETS), (y / C::Q_SETS) & 1);
        }
    } else if (wid == C::WARP_WALK) {
        if (!split_schedule(p, lane, g, runs, run_full, run_empty, [&] { return *s_abort != 0; }, p.passes, [](int) {})) give_up(1);
    } else if (wid >= C::WARP_MMA) {
        // ============================ MMA of one group's windows ============================
        const int grp = wid - C::WARP_MMA;
        const uint64_t dq0 = sdesc(s0, 16, 1024), dk0 = sdesc(s0 + C::OFF_K + grp * C::K_STAGES * C::KTILE, 16, 1024);
        SplitRun run;
        int nr = 0, ks = 0, kp = 0, job = 0, epoch = 0;  // this group's K ring and jobs
        bool ok;
        while ((ok = take_run(nr++, run)) && run.n) {
            const int n = rows_of(run), set = epoch % C::Q_SETS;
            if ((run.how & RUN_Q_NEW) && !(ok = wait(q_full + 8 * set, epoch / C::Q_SETS))) break;
            for (int x = grp; ok && x < run.n; x += 2) {
                int st[C::PARTS];  // the window's tiles; they stay until its last products are done
#pragma unroll
                for (int y = 0; y < C::PARTS; ++y) {
                    ok = ok && wait(k_full + 32 * grp + 8 * ks, kp);
                    st[y] = ks;
                    if (++ks == C::K_STAGES) ks = 0, kp ^= 1;
                }
                if (!ok) break;
                for (int r0 = 0; r0 < n; r0 += 128, ++job) {
                    const int b = 2 * grp + (job & 1), cols = min(128, n - r0);
                    if (job >= 2 && !(ok = wait(d_empty + 8 * b, (job >> 1) - 1))) break;
                    tc_fence_after();
                    const uint32_t id = idesc(bf16, 128, cols, false);
                    const uint64_t b0 = dq0 + (uint64_t)((set * C::QTILE + r0 * 128) >> 4);
#pragma unroll
                    for (int kk = 0; kk < E / 16; ++kk)
                        umma_warp(tmem + 128 * b, dk0 + (uint64_t)((st[kk / KS] * C::KTILE + ((kk % KS) >> 2) * C::KPANEL + (kk & 3) * 32) >> 4),
                                  b0 + (uint64_t)(((kk >> 2) * C::QPANEL + (kk & 3) * 32) >> 4), id, kk > 0 ? 1u : 0u);
                    umma_commit_warp(d_full + 8 * b);
                }
                if (!ok) break;
#pragma unroll
                for (int y = 0; y < C::PARTS; ++y) umma_commit_warp(k_empty + 32 * grp + 8 * st[y]);
            }
            if (!ok) break;
            if (run.how & RUN_Q_END) {
                umma_commit_warp(q_empty + 8 * set);  // arrives when this group's products of the tile are done
                ++epoch;
            }
        }
        if (!ok) give_up(2);
        // all issued MMAs have completed before TMEM is released
        umma_commit_warp(m_done + 8 * grp);
        mbar_wait(m_done + 8 * grp, 0);
    } else {
        // =============================== sums of one group's windows ===============================
        const int grp = wid >> 2, r = (wid & 3) * 32 + lane;
        const uint32_t tD = tmem + ((uint32_t)((wid & 3) * 32) << 16) + 256 * grp;
        const uint64_t sc2 = f2u(p.scale_log2, p.scale_log2);
        SplitRun run;
        int nr = 0, job = 0, epoch = 0;
        bool ok;
        while ((ok = take_run(nr++, run)) && run.n) {
            const int n = rows_of(run), set = epoch % C::Q_SETS;
            if ((run.how & RUN_Q_NEW) && !(ok = wait(q_full + 8 * set, epoch / C::Q_SETS))) break;
            const float* nlse = reinterpret_cast<const float*>(smem + C::OFF_ROW + set * C::ROWDATA);
            const int* lim = reinterpret_cast<const int*>(nlse + C::ROWS);
            const int seen_by_all = __ldcg(p.all + ((size_t)run.f * p.W + run.w) * p.Hkv + h);
            float* mrow = p.mass + ((size_t)run.w * p.Hkv + h) * p.N + run.off;
            for (int x = grp; ok && x < run.n; x += 2) {
                const int key = run.k0 + x * KT + r;
                const bool mine = key >= 0 && key < run.sp && (long long)run.off + key < p.N;
                const bool every = run.k0 + x * KT >= 0 && run.k0 + x * KT + KT <= seen_by_all;
                uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
                for (int r0 = 0; r0 < n; r0 += 128, ++job) {
                    const int b = job & 1, cols = min(128, n - r0);
                    if (!(ok = wait(d_full + 8 * (2 * grp + b), job >> 1))) break;
                    tc_fence_after();
                    auto columns = [&](float (&s)[32], int c0, int m) {  // the weights of rows c0..c0+m-1
                        const float4* nl4 = reinterpret_cast<const float4*>(nlse + c0);
                        if (every) {
#pragma unroll
                            for (int u = 0; u < 8; ++u) {
                                if (4 * u >= m) break;  // m is 16 or 32
                                const float4 nl = nl4[u];
                                float a, b2, c, d;
                                u2f(ffma2(f2u(s[4 * u], s[4 * u + 1]), sc2, f2u(nl.x, nl.y)), a, b2);
                                u2f(ffma2(f2u(s[4 * u + 2], s[4 * u + 3]), sc2, f2u(nl.z, nl.w)), c, d);
                                sum[(2 * u) & 3] = fadd2(sum[(2 * u) & 3], f2u(ex2(a), ex2(b2)));
                                sum[(2 * u + 1) & 3] = fadd2(sum[(2 * u + 1) & 3], f2u(ex2(c), ex2(d)));
                            }
                        } else {
#pragma unroll
                            for (int u = 0; u < 32; u += 2) {
                                if (u >= m) break;
                                const float a = key >= 0 && key < lim[c0 + u] ? ex2(fmaf(s[u], p.scale_log2, nlse[c0 + u])) : 0.f;
                                const float b2 = key >= 0 && key < lim[c0 + u + 1] ? ex2(fmaf(s[u + 1], p.scale_log2, nlse[c0 + u + 1])) : 0.f;
                                sum[(u >> 1) & 3] = fadd2(sum[(u >> 1) & 3], f2u(a, b2));
                            }
                        }
                    };
                    const uint32_t t = tD + 128 * b;
                    int c = 0;
                    for (; c + 64 <= cols; c += 64) {  // 64 columns in flight
                        float v0[32], v1[32];
                        tmem_ld32(t + c, v0);
                        tmem_ld32(t + c + 32, v1);
                        tmem_wait_ld();
                        reg_fence<32>(v0);
                        reg_fence<32>(v1);
                        columns(v0, r0 + c, 32);
                        columns(v1, r0 + c + 32, 32);
                    }
                    for (; c < cols; c += 32) {  // columns past the last hold an older job's scores: not used
                        float v0[32];
                        tmem_ld32(t + c, v0);
                        tmem_wait_ld();
                        reg_fence<32>(v0);
                        columns(v0, r0 + c, min(32, cols - c));
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(d_empty + 8 * (2 * grp + b));
                }
                if (!ok) break;
                float a0, a1;
                u2f(fadd2(fadd2(sum[0], sum[1]), fadd2(sum[2], sum[3])), a0, a1);
                // one addition a key and pass, by the same thread in every pass: the order is fixed, and
                // no thread waits for the old value (read by the threads: 53 instead of 36 us a decode step)
                if (mine) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(mrow + key), "f"(a0 + a1) : "memory");
            }
            if (!ok) break;
            if (run.how & RUN_Q_END) {
                __syncwarp();
                if (lane == 0) mbar_arrive(q_empty + 8 * set);
                ++epoch;
            }
        }
        if (!ok) give_up(8);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (wid == C::WARP_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <class T, int E, int ROWS> static MassKernel mass_tc() {
    using C = MassCfg<E, ROWS>;
    return MassKernel{(const void*)&mass_tc_kernel<T, E, ROWS>, C::NT, C::KT, 1, C::ROWS, (size_t)C::SMEM};
}
template <class T> static MassKernel mass_tc_e(int E, int rows) {
    // The smaller query tiles leave more of the shared memory to the K rings, the larger ones run the
    // windows fewer times: head dim 128, 128 rows 57 us with tiles of 256 rows and 61 with 512, 496
    // rows 186 and 176.
    if (E == 64) return rows <= 64 ? mass_tc<T, 64, 64>() : mass_tc<T, 64, 512>();
    if (E == 128) return rows <= 64 ? mass_tc<T, 128, 64>() : rows <= 256 ? mass_tc<T, 128, 256>() : mass_tc<T, 128, 512>();
    return rows <= 64 ? mass_tc<T, 256, 64>() : mass_tc<T, 256, 128>();
}
MassKernel mass_tc_pick(int dtype, int E, int rows) { return dtype == DVATTN_FLOAT16 ? mass_tc_e<__half>(E, rows) : mass_tc_e<__nv_bfloat16>(E, rows); }

bool mass_tc_maps(MassParams& p, int dtype, int E, MassMaps& m) {
    if (!encode_cache_map(&m.q, p.qr, dtype, E, 1, (long long)p.F * p.W * p.Hkv * p.rows_pad, 64)) return false;
    p.box = window_box(p.BS, p.kt, p.NB);
    p.align = p.box ? p.box : 1;
    return !p.box || encode_cache_map(&m.k, p.k, dtype, E, p.Hkv, p.NB * p.BS, p.box);
}

}  // namespace dvb
