// Accumulated attention weight: how much of the softmax every cached key received.
//
//   mass[w, h, off_f + l] += sum over the query heads g of KV head h and the queries s of
//   exp(scale * q_f[w, g, s] . k_l - lse[w, g, s])   for the keys that (w, s) sees,
//
// with the log-sum-exp that the attention call of the same queries returned.  A query whose
// lse is -inf (it saw nothing, or the caller takes it out) gives no weight.  Every key's sum
// is formed by one thread block in a fixed order, so results repeat bit by bit.
//
// Two launches: mass_prep_kernel (rotated queries of every turn, spans), then the kernel
// that streams the keys once.
#include "mass.cuh"

#include <cstdio>
#include <cstdlib>

namespace dvb {

// ---- prep: block (w, 16-row tile of a KV head, turn) -----------------------------------
// The queries rotated for every turn, once for all the CTAs that read them; what each row and
// every row sees of the turn; the spans.
//
// The tensor-core kernel takes a window that every counted row sees without a mask, so what a row
// without weight adds there has to vanish by itself.  Zeros with an lse of infinity would not, next to
// a key that is not finite (0 * inf).  Such a row takes the query of one that counts, its twin,
// and the most negative lse: 2^(score - most) is 0 wherever the twin's weight is finite.
constexpr int kPrepRows = 16;
constexpr float kMostFloat = 3.402823466e38f;

template <class T>
__global__ void __launch_bounds__(128) mass_prep_kernel(MassParams p, int E) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // a programmatic dependent of whatever is before it
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, f = blockIdx.z, w = blockIdx.x;
    const int tiles = p.rows_pad / kPrepRows;
    const int h = blockIdx.y / tiles, r0 = (blockIdx.y - h * tiles) * kPrepRows;
    auto row_lse = [&](int r) { return r < p.rows ? __ldg(p.lse + ((size_t)w * p.Hq + h * p.G + r % p.G) * p.S + r / p.G) : neg_inf(); };
    long long off = 0;
    for (int t = 0; t < f; ++t) off += max(__ldg(p.L + t), 0);
    const int Lf = __ldg(p.L + f);
    const size_t fw = (size_t)f * p.W + w, fwh = fw * p.Hkv + h;
    auto seen = [&](int s) { return turn_seen(Lf, __ldg(p.loc + fw * p.S + s), off, p.cap); };
    __shared__ int red[4];
    if (r0 == 0) {  // this (turn, sequence, head): what every row sees that gives weight
        int least = 0x7fffffff;
        for (int r = tid; r < p.rows; r += 128)
            if (row_lse(r) != neg_inf()) least = min(least, seen(r / p.G));
        least = __reduce_min_sync(0xffffffffu, least);
        if (lane == 0) red[tid >> 5] = least;
        __syncthreads();
        least = min(min(red[0], red[1]), min(red[2], red[3]));
        if (tid == 0) p.all[fwh] = least == 0x7fffffff ? 0 : least;
        __syncthreads();
    }
    if (blockIdx.y == 0 && f == 0) {
        if (w == 0 && tid < 4) p.header[tid] = 0;
        long long at = 0;
        int nw = 0;
        for (int t = 0; t < p.F; ++t) {
            const int Lt = __ldg(p.L + t);
            int v = 0;
            for (int s = tid; s < p.S; s += 128) v = max(v, turn_seen(Lt, __ldg(p.loc + ((size_t)t * p.W + w) * p.S + s), at, p.cap));
            v = __reduce_max_sync(0xffffffffu, v);
            if (lane == 0) red[tid >> 5] = v;
            __syncthreads();
            v = max(max(red[0], red[1]), max(red[2], red[3]));
            __syncthreads();
            const int first = v > 0 ? (int)at : 0;
            if (tid == 0) p.span[(size_t)w * p.F + t] = make_int2(v, first);
            nw += turn_windows(p, v, first);
            at += max(Lt, 0);
        }
        if (tid == 0) p.nwin[w] = nw;
    }
    if (tid < kPrepRows) {
        const int r = r0 + tid;
        const float x = row_lse(r);
        const size_t wh = (size_t)w * p.Hkv + h;
        if (f == 0) p.nlse[wh * p.rows_pad + r] = x == neg_inf() ? -kMostFloat : -x * kLog2e;
        p.lim[fwh * p.rows_pad + r] = x == neg_inf() ? 0 : seen(r / p.G);
    }
    const unsigned dead = __ballot_sync(0xffffffffu, lane < kPrepRows && row_lse(r0 + lane) == neg_inf());
    int twin = p.rows;  // the first row of the head that gives weight
    for (int b = 0; dead && b < p.rows && twin == p.rows; b += 32 * 8) {
        int first = p.rows;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (row_lse(b + 32 * u + lane) != neg_inf()) first = min(first, b + 32 * u + lane);
        twin = __reduce_min_sync(0xffffffffu, first);
    }
    constexpr int AHEAD = 2;  // chunks a thread has in flight
    const int per = E * (int)sizeof(T) / 16, n = kPrepRows * per;
    for (int c0 = tid; c0 < n; c0 += 128 * AHEAD) {
        RotateChunk<T> ch[AHEAD];
        bool counts[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const int c = c0 + 128 * k;
            counts[k] = false;
            if (c >= n) break;
            const int own = r0 + c / per, r = dead >> (own - r0) & 1u ? twin : own, s = r / p.G, e0 = c % per * RotateChunk<T>::PER;
            T* dst = static_cast<T*>(p.qr) + (fwh * p.rows_pad + own) * E;
            counts[k] = r < p.rows;
            if (counts[k])
                ch[k].load(static_cast<const T*>(p.q) + (((size_t)w * p.Hq + h * p.G + r - s * p.G) * p.S + s) * E, dst,
                           p.cos + (fw * p.S + s) * p.R, p.sin + (fw * p.S + s) * p.R, e0, p.R, p.rot_vec);
            else
                *reinterpret_cast<uint4*>(dst + e0) = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (counts[k]) ch[k].store(p.R, p.rot_vec);
    }
}

// ---- CUDA-core kernel: 32 keys x 32 rows per step, 8 warps of 4 rows, a lane per key ----
// (f32; the 16-bit types run on mass_tc_kernel)
template <int E>
__global__ void __launch_bounds__(256) mass_simt_kernel(MassParams p) {
    constexpr int KT = 32, MT = 32, ROW = E * 4 + 16, CH = E / 4;
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t* sQ = smem;                                              // [MT] rows
    uint8_t* sK = smem + MT * ROW;                                   // [KT] rows
    float* red = reinterpret_cast<float*>(sK + KT * ROW);            // [8][KT]
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int g = blockIdx.x / p.Hkv, h = blockIdx.x - g * p.Hkv;
    SplitWalk walk;
    walk.place(p, lane, g);
    SplitPiece pc;
    while (walk.next(p, pc)) {
        SplitWin win;
        win.start(p, pc.w);
        for (int i = pc.i0; i < pc.i1; ++i) {
            win.seek(p, pc.w, i);
            for (int c = tid; c < KT * CH; c += 256) {
                const int r = c / CH, ch = c - r * CH;
                const float* kp = nullptr;
                if (r < win.n) {
                    const int pos = win.off + win.k0 + r;
                    const int page = __ldg(p.bt + (size_t)pc.w * p.maxb + pos / p.BS);
                    if (page >= 0 && page < p.NB)
                        kp = static_cast<const float*>(p.k) + (((size_t)page * p.BS + pos % p.BS) * p.Hkv + h) * E + ch * 4;
                }
                cp_async16_zfill(smem_u32(sK + r * ROW + ch * 16), kp ? kp : static_cast<const float*>(p.k), kp ? 16 : 0);
            }
            cp_async_commit();
            const float* qr = static_cast<const float*>(p.qr) + (((size_t)win.f * p.W + pc.w) * p.Hkv + h) * p.rows_pad * E;
            const float* nlse = p.nlse + ((size_t)pc.w * p.Hkv + h) * p.rows_pad;
            const int* lim = p.lim + (((size_t)win.f * p.W + pc.w) * p.Hkv + h) * p.rows_pad;
            float acc = 0.f;
            for (int r0 = 0; r0 < p.rows; r0 += MT) {
                for (int c = tid; c < MT * CH; c += 256) {
                    const int r = c / CH, ch = c - r * CH;
                    const bool in = r0 + r < p.rows;
                    cp_async16_zfill(smem_u32(sQ + r * ROW + ch * 16), qr + (size_t)(in ? r0 + r : 0) * E + ch * 4, in ? 16 : 0);
                }
                cp_async_commit();
                cp_async_wait<0>();
                __syncthreads();
                float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                for (int ch = 0; ch < CH; ++ch) {
                    const float4 k4 = *reinterpret_cast<const float4*>(sK + lane * ROW + ch * 16);
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const float4 q4 = *reinterpret_cast<const float4*>(sQ + (wid * 4 + a) * ROW + ch * 16);
                        sc[a] = fmaf(q4.x, k4.x, sc[a]);
                        sc[a] = fmaf(q4.y, k4.y, sc[a]);
                        sc[a] = fmaf(q4.z, k4.z, sc[a]);
                        sc[a] = fmaf(q4.w, k4.w, sc[a]);
                    }
                }
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const int r = r0 + wid * 4 + a;
                    if (r >= p.rows) continue;
                    if (lane < win.n && win.k0 + lane < __ldcg(lim + r)) acc += fast_exp2(fmaf(sc[a], p.scale_log2, __ldcg(nlse + r)));
                }
                __syncthreads();
            }
            red[wid * KT + lane] = acc;
            __syncthreads();
            if (wid == 0 && lane < win.n) {
                const long long pos = (long long)win.off + win.k0 + lane;
                if (pos < p.N) {
                    float sum = red[lane];
#pragma unroll
                    for (int x = 1; x < 8; ++x) sum += red[x * KT + lane];
                    p.mass[((size_t)pc.w * p.Hkv + h) * p.N + pos] += sum;
                }
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------------------
template <int E> static MassKernel mass_simt() {
    const size_t smem = (size_t)64 * (E * 4 + 16) + 8 * 32 * 4;
    return MassKernel{(const void*)&mass_simt_kernel<E>, 256, 32, E == 64 ? 8 : E == 128 ? 6 : 3, 1 << 30, smem};
}
static MassKernel mass_pick(const dvattn_mass_args* a) {
    if (a->dtype != DVATTN_FLOAT32) return mass_tc_pick(a->dtype, a->E, a->S * (a->Hq / a->Hkv));
    return a->E == 64 ? mass_simt<64>() : a->E == 128 ? mass_simt<128>() : mass_simt<256>();
}

// DVATTN_TEST_STALL_TILE=<i>: tests only (see the decode launcher); read once per process.
static int mass_stall_hook() {
    static const int t = [] {
        const char* e = getenv("DVATTN_TEST_STALL_TILE");
        return e && *e ? atoi(e) : -1;
    }();
    return t;
}
static long long mass_rows_pad(const dvattn_mass_args* a) { return ((long long)a->S * (a->Hq / a->Hkv) + kPrepRows - 1) / kPrepRows * kPrepRows; }

static int mass_validate(const dvattn_mass_args* a) {
    if (!a) return DVATTN_ERR_INVALID_ARGUMENT;
    dvattn_paged_args v{};  // the shape rules of the paged attention
    v.dtype = a->dtype; v.F = a->F; v.W = a->W; v.Hq = a->Hq; v.Hkv = a->Hkv; v.E = a->E; v.Ev = a->E; v.S = a->S;
    v.R = a->R; v.block_size = a->block_size; v.max_blocks_per_seq = a->max_blocks_per_seq; v.num_blocks = a->num_blocks;
    const int st = decode_validate(&v);
    if (st != DVATTN_OK) return st;
    if (a->positions < 0) return DVATTN_ERR_INVALID_ARGUMENT;
    // grid limits of the prep kernel: turns are its z, row tiles of the KV heads its y; 32-bit rows
    if (a->F > 65535 || mass_rows_pad(a) / kPrepRows * a->Hkv > 65535 || (double)a->F * a->W * a->Hkv * mass_rows_pad(a) > 0x7fffffffLL - 128)
        return DVATTN_ERR_UNSUPPORTED;
    return DVATTN_OK;
}
static bool mass_nothing(const dvattn_mass_args* a) {
    return (long long)a->W * a->S == 0 || a->Hq == 0 || a->F == 0 || a->positions == 0 || a->num_blocks <= 0 || a->max_blocks_per_seq == 0;
}

struct MassLayout {
    size_t nwin, span, qr, nlse, lim, all, total;
    int groups;
};
static int mass_layout(const dvattn_mass_args* a, const MassKernel& k, MassLayout& L) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
        cudaFuncSetAttribute(k.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem) != cudaSuccess)
        return DVATTN_ERR_CUDA;
    L.groups = sms * k.ctas / a->Hkv;
    if (L.groups < 1) L.groups = 1;
    const size_t esz = a->dtype == DVATTN_FLOAT32 ? 4 : 2, rows = (size_t)mass_rows_pad(a), wh = (size_t)a->W * a->Hkv;
    size_t at = 256;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    L.nwin = take(4 * (size_t)a->W);
    L.span = take(8 * (size_t)a->W * a->F);
    L.qr = take(esz * a->F * wh * rows * a->E);
    L.nlse = take(4 * wh * rows);
    L.lim = take(4 * a->F * wh * rows);
    L.all = take(4 * a->F * wh);
    L.total = at;
    return DVATTN_OK;
}

size_t mass_workspace_size(const dvattn_mass_args* a) {
    if (mass_validate(a) != DVATTN_OK || mass_nothing(a)) return 0;
    MassLayout L;
    return mass_layout(a, mass_pick(a), L) == DVATTN_OK ? L.total : 0;
}

int mass_launch(const dvattn_mass_args* a, void* workspace, size_t wbytes, cudaStream_t stream) {
    int st = mass_validate(a);
    if (st != DVATTN_OK) return st;
    if (mass_nothing(a)) return DVATTN_OK;
    if (!a->mass || !a->queries || !a->lse || !a->locations || !a->fragment_lengths || !a->k_cache || !a->block_tables ||
        (a->R > 0 && (!a->cosines || !a->sines)))
        return DVATTN_ERR_INVALID_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(a->queries) & 15) || (reinterpret_cast<uintptr_t>(a->k_cache) & 15)) return DVATTN_ERR_INVALID_ARGUMENT;
    const MassKernel k = mass_pick(a);
    MassLayout L;
    if ((st = mass_layout(a, k, L)) != DVATTN_OK) return st;
    if (!workspace || wbytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return DVATTN_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    MassParams p{};
    p.F = a->F; p.W = a->W; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv; p.S = a->S; p.R = a->R;
    p.rows = p.S * p.G;
    p.rows_pad = (int)mass_rows_pad(a);
    p.passes = (p.rows_pad + k.pass_rows - 1) / k.pass_rows;
    p.stall_tile = mass_stall_hook();
    p.rot_vec = rotate_vec(a->R, a->cosines, a->sines);
    p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.NB = a->num_blocks;
    const long long cap = (long long)a->max_blocks_per_seq * a->block_size;
    p.cap = cap > kMostPositions ? kMostPositions : (int)cap;
    p.tail = 0; p.align = 1; p.kt = k.kt; p.nt = 1; p.groups = L.groups; p.least = 1;
    p.N = a->positions;
    p.scale_log2 = a->scale * kLog2e;
    p.mass = a->mass; p.lse = a->lse; p.q = a->queries; p.cos = a->cosines; p.sin = a->sines; p.k = a->k_cache;
    p.loc = a->locations; p.L = a->fragment_lengths; p.bt = a->block_tables;
    p.header = reinterpret_cast<int*>(ws);
    p.nwin = reinterpret_cast<int*>(ws + L.nwin);
    p.span = reinterpret_cast<int2*>(ws + L.span);
    p.qr = ws + L.qr;
    p.nlse = reinterpret_cast<float*>(ws + L.nlse);
    p.lim = reinterpret_cast<int*>(ws + L.lim);
    p.all = reinterpret_cast<int*>(ws + L.all);
    alignas(64) MassMaps maps;
    if (a->dtype != DVATTN_FLOAT32 && !mass_tc_maps(p, a->dtype, a->E, maps)) return DVATTN_ERR_CUDA;
    const void* prep = a->dtype == DVATTN_FLOAT32   ? (const void*)&mass_prep_kernel<float>
                       : a->dtype == DVATTN_FLOAT16 ? (const void*)&mass_prep_kernel<__half> : (const void*)&mass_prep_kernel<__nv_bfloat16>;
    int E = a->E;
    void* pargs[] = {&p, &E};
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = stream;
    cfg.gridDim = dim3(a->W, (unsigned)(p.rows_pad / kPrepRows * a->Hkv), a->F);
    cfg.blockDim = dim3(128);
    cudaError_t e = cudaLaunchKernelExC(&cfg, prep, pargs);
    if (e == cudaSuccess) {
        cfg.gridDim = dim3((unsigned)(L.groups * a->Hkv));
        cfg.blockDim = dim3(k.threads);
        cfg.dynamicSmemBytes = k.smem;
        void* args[] = {&p, &maps};  // the CUDA-core kernel takes the first only
        e = cudaLaunchKernelExC(&cfg, k.fn, args);
    }
    if (e != cudaSuccess) {
        if (getenv("DVATTN_DEBUG")) fprintf(stderr, "dvattn mass launch: %s\n", cudaGetErrorString(e));
        return DVATTN_ERR_CUDA;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
