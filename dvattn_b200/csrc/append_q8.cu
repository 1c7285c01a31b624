// Append of new tokens to a paged cache held in 8 bits (q8.cuh), keys rotated as the paged append rotates
// them (append.cu).
//
// A tile is what a call writes of one page, KV head and tensor: tokens [a, b) of the page.  With m = max |x|
// over the tile's finite elements, need = 2^ceil(log2(m / 448)), at least 2^-60; the page's scale becomes
// need where the tile begins the page (a = 0), else max(scale, need), and where it grows, the tokens [0, a)
// are stored again in the new scale.  A power of two costs e4m3 no precision (it has its own exponent) and
// makes storing again exact, but for elements that fall under its smallest normal value.
//
// A warp per tile whose groups of 8 elements its lanes can hold (kHeld each, as they are in memory), a block of four warps for
// larger ones; what a thread cannot hold it reads again (from L1) once the scale is known.  Prompts of up to 2048 tokens of 16
// sequences in pages of 16 (256 groups a tile), bf16, 2 KV heads of 128: 12.9 us with a warp per tile, 25.6 with a block (replayed
// from a graph; a call by itself takes 14.3).
//
// What bounds it is not HBM (27 MB take 4.2 us) but the length of a tile's chain, position -> page -> scale -> store, and the
// instructions of the rotation: so a tile's rotating groups come first and its other groups after them, a warp does one or
// the other, all loads of a thread are under way before the first is used, and maxima are taken of the bits, two elements an
// operation (non-finite elements have a path of their own).  32 sequences of up to 501 tokens in pages of 64, f16, 8 KV
// heads, all of 128 dims rotated: 29 us replayed, 33 by itself (63 MB), with every head reading the angles again from L2.
#include "decode.cuh"
#include "q8.cuh"
#include "tcgen05.cuh"

namespace dvb {

struct AppendQ8Params {
    int W, Hkv, E, Ev, n, R, BS, maxb;
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

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }
// x / s; a power of two is divided by exactly with a product
__device__ __forceinline__ float over(float x, float s, float inv, bool pow2) { return pow2 ? x * inv : __fdiv_rn(x, s); }

// 8 elements as they are in memory.
template <class T> struct Group {
    static constexpr int N = 2 * sizeof(T);
    uint32_t w[N];
    __device__ __forceinline__ void load(const T* x) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(x) + i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::to_f(reinterpret_cast<const T*>(w)[i]);
    }
    __device__ __forceinline__ void put(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<T*>(w)[i] = Elem<T>::from_f(v[i]);
    }
    // bits of the largest magnitude so far (16-bit types: of each half); those of an infinity, of a NaN lie above
    __device__ __forceinline__ uint32_t top(uint32_t m) const {
#pragma unroll
        for (int i = 0; i < N; ++i) m = sizeof(T) == 4 ? max(m, w[i] & 0x7fffffffu) : __vmaxu2(m, w[i] & 0x7fff7fffu);
        return m;
    }
    __device__ __forceinline__ uint64_t pair(int i) const {  // elements 2i, 2i + 1 in 32 bits
        if constexpr (sizeof(T) == 4) return f2u(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else return f2u(Elem<T>::to_f(reinterpret_cast<const T*>(w)[2 * i]), Elem<T>::to_f(reinterpret_cast<const T*>(w)[2 * i + 1]));
    }
    // These elements rotated with their partners y (a lower half's: sign set) by angles c and s, as rotated8 does it.  (The packed
    // f32x2 product and sum get contracted to a fused one, which rounds once.)
    __device__ __forceinline__ void rotate(const Group& y, const Group<float>& c, const Group<float>& s, uint32_t sign) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Group z;
#pragma unroll
            for (int k = i * N / 4; k < (i + 1) * N / 4; ++k) z.w[k] = y.w[k] ^ sign;
            float a[2], b[2];
            u2f(pair(i), a[0], a[1]);
            u2f(z.pair(i), b[0], b[1]);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                a[k] = __fadd_rn(__fmul_rn(a[k], __uint_as_float(c.w[2 * i + k])), __fmul_rn(b[k], __uint_as_float(s.w[2 * i + k])));
            if constexpr (sizeof(T) == 4) w[2 * i] = __float_as_uint(a[0]), w[2 * i + 1] = __float_as_uint(a[1]);
            else w[i] = Elem<T>::pack2(a[0], a[1]);
        }
    }
    static __device__ __forceinline__ float value(uint32_t m) {  // of those bits
        if (sizeof(T) == 4) return __uint_as_float(m);
        const unsigned short h = (unsigned short)max(m & 0xffffu, m >> 16);
        return Elem<T>::to_f(*reinterpret_cast<const T*>(&h));
    }
};

template <class T> constexpr int kHeld = 32 / Group<T>::N;  // groups that a thread holds

// i / d, i below `upto`: one product where it is exact (i (2^32 - m d) < 2^32, and m d - 2^32 < d)
struct Divide {
    unsigned d, m;
    __device__ __forceinline__ Divide(int by, int upto) : d(by), m(by > 1 && (long long)upto * by < (1LL << 32) ? 0xffffffffu / (unsigned)by + 1 : 0) {}
    __device__ __forceinline__ int operator()(int i) const { return m ? (int)__umulhi((unsigned)i, m) : d > 1 ? (int)((unsigned)i / d) : i; }
};

template <class T, int TEAM, bool VEC>  // threads of a tile: 32 or 128; whole groups of 8 rotate (see rotated8)
__global__ void __launch_bounds__(128) append_q8_kernel(AppendQ8Params p) {
    constexpr int KEEP = kHeld<T>;
    __shared__ float part[4];
    const int lane = threadIdx.x & 31, me = TEAM == 32 ? lane : threadIdx.x;
    const unsigned all = (unsigned)p.W * p.tiles * p.Hkv * 2, task = TEAM == 32 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (task >= all) return;
    const bool is_k = !(task & 1);
    const int wj = (int)((task >> 1) / p.Hkv), h = (int)((task >> 1) - (unsigned)wj * p.Hkv), w = wj / p.tiles, j = wj - w * p.tiles;
    const long long p0 = __ldg(p.pos + w);
    const int given = p.cnt ? __ldg(p.cnt + w) : p.n, cnt = given < 0 ? 0 : given < p.n ? given : p.n;
    const long long from = p0 > 0 ? p0 : 0;
    const long long pg = (int)from / p.BS + j;  // page of the table
    if (pg >= p.maxb) return;
    const long long base = pg * p.BS;
    const long long lo = from > base ? from : base, hi = p0 + cnt < base + p.BS ? p0 + cnt : base + p.BS;
    if (lo >= hi) return;
    const int page = __ldg(p.bt + (size_t)w * p.maxb + pg);
    const int a = (int)(lo - base), tokens = (int)(hi - lo);
    const int t0 = p.n - cnt + (int)(lo - p0);  // row of the first of them (left padding in front)
    const int E = is_k ? p.E : p.Ev, per = E >> 3, items = tokens * per;
    const T* x = static_cast<const T*>(is_k ? p.keys : p.values) + (((size_t)w * p.Hkv + h) * p.n + t0) * E;
    const size_t angles = ((size_t)w * p.n + t0) * p.R;
    // The tile's groups: first those that rotate, of all its tokens, then the others (warps do one or the other).
    const int turned = is_k ? (p.R + 7) >> 3 : 0, straight = per - turned, bound = tokens * turned;
    const Divide by_turned(turned, bound), by_straight(straight, items - bound);
    struct At {
        int it, tok, e0;
    };
    auto at = [&](int it) {
        const bool r = it < bound;
        const int i = r ? it : it - bound, tok = r ? by_turned(i) : by_straight(i);
        return At{it, tok, (r ? i - tok * turned : i - tok * straight + turned) << 3};
    };
    // `group` as it came from memory: rotated, where it does
    auto turn = [&](const At& g, Group<T>& group) {
        const T* row = x + (size_t)g.tok * E;
        const float *cr = p.cos + angles + (size_t)g.tok * p.R, *sr = p.sin + angles + (size_t)g.tok * p.R;
        if constexpr (VEC) {
            const int half = p.R >> 1;
            const bool lo = g.e0 < half;
            Group<T> y;
            Group<float> c, s;
            y.load(row + (lo ? g.e0 + half : g.e0 - half));
            c.load(cr + g.e0);
            s.load(sr + g.e0);
            group.rotate(y, c, s, lo ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u);
        } else {
            float y[8];
            rotated8<T, true>(row, cr, sr, g.e0, p.R, false, y);
            group.put(y);
        }
    };
    auto compute = [&](const At& g, Group<T>& group) {
        group.load(x + (size_t)g.tok * E + g.e0);
        if (g.it < bound) turn(g, group);
    };
    Group<T> keep[KEEP];
#pragma unroll
    for (int k = 0; k < KEEP; ++k) {
        const At g = at(me + k * TEAM);
        if (g.it < items) keep[k].load(x + (size_t)g.tok * E + g.e0);
    }
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
        if (me + k * TEAM < bound) turn(at(me + k * TEAM), keep[k]);
    // what the values wait for is under way: now the page
    if (page < 0 || page >= p.NB) return;
    float* sp = (is_k ? p.ks : p.vs) + (size_t)page * p.Hkv + h;
    const float old = a ? *sp : 0.f;
    uint8_t* dst = (is_k ? p.kc : p.vc) + ((size_t)page * p.BS * p.Hkv + h) * E;  // token i: + i Hkv E
    const size_t stride = (size_t)p.Hkv * E;
    auto reduced = [&](float m) {  // maximum over the team; m >= 0: the bits are in order
        m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));
        if (TEAM > 32) {
            __syncthreads();
            if (lane == 0) part[threadIdx.x >> 5] = m;
            __syncthreads();
            m = __uint_as_float(max(max(__float_as_uint(part[0]), __float_as_uint(part[1])), max(__float_as_uint(part[2]), __float_as_uint(part[3]))));
        }
        return m;
    };
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
        if (me + k * TEAM < items) bits = keep[k].top(bits);
    for (int it = me + KEEP * TEAM; it < items; it += TEAM) {
        Group<T> v;
        compute(at(it), v);
        bits = v.top(bits);
    }
    float m = reduced(Group<T>::value(bits));
    const bool odd = !finite(m);  // of the whole team: some element is not finite
    if (odd) {                    // the largest of the others
        m = 0.f;
#pragma unroll 1
        for (int it = me; it < items; it += TEAM) {
            Group<T> g;
            float v[8];
            compute(at(it), g);
            g.get(v);
#pragma unroll
            for (int u = 0; u < 8; ++u) m = fmaxf(m, finite(v[u]) ? fabsf(v[u]) : 0.f);
        }
        m = reduced(m);
    }
    // m = 1.f 2^(ex - 127) and 448 = 1.75 2^8
    const int mb = __float_as_int(m), ex = (mb >> 23) - 135 + ((mb & 0x7fffff) > 0x600000);
    const float need = __int_as_float(((ex < -60 ? -60 : ex) + 127) << 23);
    const float s = a && old > need ? old : need;
    const bool pow2 = (__float_as_int(s) & 0x7fffff) == 0 && s < 0x1p126f;
    const float inv = 1.f / s;
    if (a && old < s) {  // the tokens in front, in the new scale
        for (int it = me; it < a * per; it += TEAM) {
            const int tok = it / per;
            uint2* to = reinterpret_cast<uint2*>(dst + tok * stride + ((it - tok * per) << 3));
            uint2 q = *to;
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
            *to = q;
        }
    }
    auto put = [&](const At& g, const float (&v)[8]) {
        uint32_t q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = f32x2_to_e4m3x2(v[2 * u], v[2 * u + 1]);
        *reinterpret_cast<uint2*>(dst + (a + g.tok) * stride + g.e0) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
    };
    if (pow2 && !odd) {
        auto store = [&](const At& g, const Group<T>& group) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 4; ++u) u2f(fmul2(group.pair(u), f2u(inv, inv)), v[2 * u], v[2 * u + 1]);
            put(g, v);
        };
#pragma unroll
        for (int k = 0; k < KEEP; ++k)
            if (me + k * TEAM < items) store(at(me + k * TEAM), keep[k]);
        for (int it = me + KEEP * TEAM; it < items; it += TEAM) {
            Group<T> v;
            compute(at(it), v);
            store(at(it), v);
        }
    } else {
#pragma unroll 1
        for (int it = me; it < items; it += TEAM) {
            Group<T> group;
            float v[8];
            compute(at(it), group);
            group.get(v);
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = finite(v[u]) ? over(v[u], s, inv, pow2) : __int_as_float(0x7fc00000);  // NaN: an infinity, too
            put(at(it), v);
        }
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
    const long long groups = (long long)(a->n < a->block_size ? a->n : a->block_size) * (a->E > a->Ev ? a->E : a->Ev) / 8;
    const bool vec = a->R % 16 == 0 && !((reinterpret_cast<uintptr_t>(a->cosines) | reinterpret_cast<uintptr_t>(a->sines)) & 15);
    auto go = [&](auto zero) {
        using T = decltype(zero);
        const bool small = groups <= 32 * kHeld<T>;
        const unsigned grid = (unsigned)(small ? (all + 3) / 4 : all);
        auto* fn = small ? (vec ? append_q8_kernel<T, 32, true> : append_q8_kernel<T, 32, false>)
                         : (vec ? append_q8_kernel<T, 128, true> : append_q8_kernel<T, 128, false>);
        fn<<<grid, 128, 0, stream>>>(p);
    };
    switch (a->dtype) {
        case DVATTN_FLOAT16: go(__half()); break;
        case DVATTN_BFLOAT16: go(__nv_bfloat16()); break;
        default: go(float()); break;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

}  // namespace dvb
