// Append of new tokens to a paged cache held in 8 bits (q8.cuh), keys rotated as the paged append rotates
// them (append.cu).
//
// A tile is what a call writes of one page, KV head and tensor: tokens [a, b) of the page.  With m = max |x|
// over the tile's finite elements, need = 2^ceil(log2(m / 448)), at least 2^-60; the page's scale becomes
// need where the tile begins the page (a = 0), else max(scale, need), and where it grows, the tokens [0, a)
// are stored again in the new scale.  A power of two costs e4m3 no precision (it has its own exponent) and
// makes storing again exact, but for elements that fall under its smallest normal value.
//
// A warp per tile where it has few elements (decode steps), a block of four warps otherwise.  A thread holds
// the first kKeep groups of 8 elements it computed and reads those past them again (from L1) once the
// scale is known.
#include "decode.cuh"
#include "q8.cuh"

namespace dvb {

struct AppendQ8Params {
    int W, Hkv, E, Ev, n, R, BS, maxb;
    int vec;    // see rotated8
    int tiles;  // pages that n tokens of a worker can touch
    long long NB;
    uint8_t* kc;
    uint8_t* vc;
    float* ks;
    float* vs;
    const void* keys;
    const void* values;
    const float* cos;
    const float* sin;
    const int* bt;
    const int* pos;
    const int* cnt;
};

constexpr int kKeep = 4;

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }
// x / s; a power of two is divided by exactly with a product
__device__ __forceinline__ float over(float x, float s, float inv, bool pow2) { return pow2 ? x * inv : __fdiv_rn(x, s); }

template <class T, int TEAM>  // threads of a tile: 32 or 128
__global__ void __launch_bounds__(128) append_q8_kernel(AppendQ8Params p) {
    __shared__ float part[4];
    const int lane = threadIdx.x & 31, me = TEAM == 32 ? lane : threadIdx.x;
    const long long task = TEAM == 32 ? (long long)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (task >= (long long)p.W * p.tiles * p.Hkv * 2) return;
    const bool is_k = !(task & 1);
    const int wj = (int)((task >> 1) / p.Hkv), h = (int)((task >> 1) - (long long)wj * p.Hkv), w = wj / p.tiles, j = wj - w * p.tiles;
    const long long p0 = __ldg(p.pos + w);
    const int given = p.cnt ? __ldg(p.cnt + w) : p.n, cnt = given < 0 ? 0 : given < p.n ? given : p.n;
    const long long from = p0 > 0 ? p0 : 0;
    const long long pg = from / p.BS + j;  // page of the table
    if (pg >= p.maxb) return;
    const long long base = pg * p.BS;
    const long long lo = from > base ? from : base, hi = p0 + cnt < base + p.BS ? p0 + cnt : base + p.BS;
    if (lo >= hi) return;
    const int page = __ldg(p.bt + (size_t)w * p.maxb + pg);
    if (page < 0 || page >= p.NB) return;
    const int a = (int)(lo - base), tokens = (int)(hi - lo);
    const int t0 = p.n - cnt + (int)(lo - p0);  // row of the first of them (left padding in front)
    const int E = is_k ? p.E : p.Ev, per = E >> 3, items = tokens * per;
    float* sp = (is_k ? p.ks : p.vs) + (size_t)page * p.Hkv + h;
    const float old = a ? *sp : 0.f;
    const T* x = static_cast<const T*>(is_k ? p.keys : p.values) + (((size_t)w * p.Hkv + h) * p.n + t0) * E;
    const size_t angles = ((size_t)w * p.n + t0) * p.R;
    uint8_t* dst = (is_k ? p.kc : p.vc) + ((size_t)page * p.BS * p.Hkv + h) * E;  // token i: + i Hkv E
    const size_t stride = (size_t)p.Hkv * E;
    auto compute = [&](int it, float (&v)[8]) {
        const int tok = it / per, e0 = (it - tok * per) << 3;
        const T* row = x + (size_t)tok * E;
        if (is_k) rotated8<T, true>(row, p.cos + angles + (size_t)tok * p.R, p.sin + angles + (size_t)tok * p.R, e0, p.R, p.vec, v);
        else load8(row + e0, v);
    };
    float keep[kKeep][8];
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
        const int it = me + k * TEAM;
        if (it < items) compute(it, keep[k]);
    }
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
        if (me + k * TEAM < items)
#pragma unroll
            for (int u = 0; u < 8; ++u) m = fmaxf(m, finite(keep[k][u]) ? fabsf(keep[k][u]) : 0.f);
    for (int it = me + kKeep * TEAM; it < items; it += TEAM) {
        float v[8];
        compute(it, v);
#pragma unroll
        for (int u = 0; u < 8; ++u) m = fmaxf(m, finite(v[u]) ? fabsf(v[u]) : 0.f);
    }
    m = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(m)));  // m >= 0: the bits are in order
    if (TEAM > 32) {
        if (lane == 0) part[threadIdx.x >> 5] = m;
        __syncthreads();
        m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    }
    // m = 1.f 2^(ex - 127) and 448 = 1.75 2^8
    const int bits = __float_as_int(m), ex = (bits >> 23) - 135 + ((bits & 0x7fffff) > 0x600000);
    const float need = __int_as_float(((ex < -60 ? -60 : ex) + 127) << 23);
    const float s = a && old > need ? old : need;
    const bool pow2 = (__float_as_int(s) & 0x7fffff) == 0 && s < 0x1p126f;
    const float inv = 1.f / s;
    if (a && old < s) {  // the tokens in front, in the new scale
        for (int it = me; it < a * per; it += TEAM) {
            const int tok = it / per;
            uint2* at = reinterpret_cast<uint2*>(dst + tok * stride + ((it - tok * per) << 3));
            uint2 q = *at;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t& word = u ? q.y : q.x;
                uint32_t out = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint32_t f = e4m3x2_to_f16x2(word >> (16 * b) & 0xffffu);
                    const __half2 f2 = *reinterpret_cast<const __half2*>(&f);
                    out |= f32x2_to_e4m3x2(over(__fmul_rn(__low2float(f2), old), s, inv, pow2), over(__fmul_rn(__high2float(f2), old), s, inv, pow2)) << (16 * b);
                }
                word = out;
            }
            *at = q;
        }
    }
    auto store = [&](int it, const float (&v)[8]) {
        const int tok = it / per, e0 = (it - tok * per) << 3;
        uint32_t q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float nan = __int_as_float(0x7fc00000);  // an infinity, too
            const float y0 = finite(v[2 * u]) ? over(v[2 * u], s, inv, pow2) : nan, y1 = finite(v[2 * u + 1]) ? over(v[2 * u + 1], s, inv, pow2) : nan;
            q[u] = f32x2_to_e4m3x2(y0, y1);
        }
        *reinterpret_cast<uint2*>(dst + (a + tok) * stride + e0) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
    };
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
        if (me + k * TEAM < items) store(me + k * TEAM, keep[k]);
    for (int it = me + kKeep * TEAM; it < items; it += TEAM) {
        float v[8];
        compute(it, v);
        store(it, v);
    }
    if (me == 0) *sp = s;  // everyone has read the old one (the reduction lies between)
}

int append_q8_launch(const dvattn_append_args* a, const dvattn_q8_scales* sc, cudaStream_t stream) {
    if (!a || !sc) return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->dtype < 0 || a->dtype > 2) return DVATTN_ERR_UNSUPPORTED;
    if (a->W < 0 || a->n < 0 || a->Hkv <= 0 || a->E <= 0 || a->Ev <= 0 || a->R < 0 || a->R > a->E || (a->R & 1) || a->block_size <= 0 ||
        a->max_blocks_per_seq < 0 || a->num_blocks < 0)
        return DVATTN_ERR_INVALID_ARGUMENT;
    if (a->E % 8 || a->Ev % 8) return DVATTN_ERR_UNSUPPORTED;
    if ((long long)a->W * a->n == 0) return DVATTN_OK;
    const long long tiles = ((long long)a->n + a->block_size - 2) / a->block_size + 1, all = (long long)a->W * tiles * a->Hkv * 2;
    // tokens x groups of a tile, tiles (a grid's blocks) and positions are counted in 32 bits
    if ((long long)a->W * a->n >= (1LL << 31) || (long long)a->max_blocks_per_seq * a->block_size >= (1LL << 31) ||
        (long long)a->block_size * (a->E > a->Ev ? a->E : a->Ev) >= (1LL << 31) || (long long)a->W * tiles >= (1LL << 31) || all >= (1LL << 31))
        return DVATTN_ERR_UNSUPPORTED;
    if (!a->k_cache || !a->v_cache || !sc->k_scales || !sc->v_scales || !a->keys || !a->values || !a->block_tables || !a->positions ||
        (a->R > 0 && (!a->cosines || !a->sines)))
        return DVATTN_ERR_INVALID_ARGUMENT;
    for (const void* q : {(const void*)a->k_cache, (const void*)a->v_cache, a->keys, a->values})
        if (reinterpret_cast<uintptr_t>(q) & 15) return DVATTN_ERR_INVALID_ARGUMENT;
    AppendQ8Params p{};
    p.W = a->W; p.Hkv = a->Hkv; p.E = a->E; p.Ev = a->Ev; p.n = a->n; p.R = a->R; p.BS = a->block_size; p.maxb = a->max_blocks_per_seq;
    p.NB = a->num_blocks; p.tiles = (int)tiles;
    p.kc = static_cast<uint8_t*>(a->k_cache); p.vc = static_cast<uint8_t*>(a->v_cache);
    p.ks = sc->k_scales; p.vs = sc->v_scales; p.keys = a->keys; p.values = a->values;
    p.cos = a->cosines; p.sin = a->sines; p.bt = a->block_tables; p.pos = a->positions; p.cnt = a->counts;
    p.vec = a->R % 16 == 0 && !((reinterpret_cast<uintptr_t>(a->cosines) | reinterpret_cast<uintptr_t>(a->sines)) & 15);
    const long long groups = (long long)(a->n < a->block_size ? a->n : a->block_size) * (a->E > a->Ev ? a->E : a->Ev) / 8;
    const bool small = groups <= 2 * 32;
    const unsigned grid = (unsigned)(small ? (all + 3) / 4 : all);
    auto go = [&](auto* one, auto* four) {
        if (small) one<<<grid, 128, 0, stream>>>(p);
        else four<<<grid, 128, 0, stream>>>(p);
    };
    switch (a->dtype) {
        case DVATTN_FLOAT16: go(&append_q8_kernel<__half, 32>, &append_q8_kernel<__half, 128>); break;
        case DVATTN_BFLOAT16: go(&append_q8_kernel<__nv_bfloat16, 32>, &append_q8_kernel<__nv_bfloat16, 128>); break;
        default: go(&append_q8_kernel<float, 32>, &append_q8_kernel<float, 128>); break;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
