// Work split over the cached turns of a batch, shared by the kernels in which all query rows
// of a sequence's KV head read the same keys (tree.cu, tree_tc.cu, mass.cu).
//
// A sequence's keys are cut into windows of `kt` keys: each turn's visible keys (the union
// over the queries) from the turn's first key on (or from up to `align` - 1 positions before
// it, so that windows begin on a multiple of `align`), then `tail` keys that lie outside the
// cache (the drafted tokens of a tree; 0 where there are none).  The windows of all
// (sequence, row tile) pairs, one after the other, are cut into `groups` ranges of equal
// length.  A group is Hkv CTAs that walk the same range, one KV head each, so the heads of a
// token (contiguous in a page) are read at about the same time.
#pragma once

#include "tcgen05.cuh"
#include "decode.cuh"

namespace dvb {

// Positions of a sequence that are read at most: window arithmetic reaches up to two windows past the
// last key, and stays within 32 bits.
constexpr int kMostPositions = 0x7fffff00;

struct TurnSplit {
    int F, W, BS, maxb, cap, tail;  // cap: positions of the block table, at most kMostPositions
    int kt, nt, groups;  // keys per window, row tiles per sequence, CTA groups
    int least;           // windows a group has at least, where there are that many
    int align;           // windows over the cache begin on logical positions that are multiples of it
    long long NB;
    const int* loc;
    const int* L;
    const int* bt;
    int* nwin;  // workspace: [W] windows of a sequence's row tile
    // workspace: [W][F] {keys of the turn that some query of the sequence sees, its first position}; the
    // sign bit of the position: another query does not see them all (where the kernel asks for it)
    int2* span;
};

// Keys of a turn that a query with location `loc` sees, the turn starting at logical
// position `off`: l <= loc, l < L and off + l < cap.
__device__ __forceinline__ int turn_seen(int L, int loc, long long off, int cap) {
    if (loc < 0 || L <= 0 || off >= cap) return 0;
    const int v = loc >= L ? L : loc + 1;
    const long long room = cap - off;
    return v < room ? v : (int)room;
}

// Windows of a turn of which `seen` keys are seen (`align` is a power of two).
__device__ __forceinline__ int turn_windows(const TurnSplit& p, int seen, int off) {
    return seen > 0 ? ((off & (p.align - 1)) + seen + p.kt - 1) / p.kt : 0;
}

// The split of `total` windows over the groups that get any (every one at least p.least, so that
// short calls do not fall into more partial results than the merge is quick with): the first
// total % groups of them take one window more than the others.
struct SplitRange {
    long long q, r;  // windows of a group, groups with one more
    int groups;
    __device__ __forceinline__ SplitRange(long long total, const TurnSplit& p) {
        const long long most = total / p.least;
        groups = most < p.groups ? (most > 0 ? (int)most : 1) : p.groups;
        if (total <= 0x7fffffffLL) {
            const unsigned t = (unsigned)total, n = (unsigned)groups;
            q = t / n;
            r = t % n;
        } else {
            q = total / groups;
            r = total % groups;
        }
    }
    __device__ __forceinline__ long long begin(int g) const {
        if (g > groups) g = groups;
        return g * q + (g < r ? g : r);
    }
    // the group of window u < total; the groups between two windows' are never empty
    __device__ __forceinline__ int group_of(long long u) const {
        const long long more = r * (q + 1);
        if (u < more) return (int)(u <= 0x7fffffffLL && q < 0x7fffffffLL ? (unsigned)u / (unsigned)(q + 1) : u / (q + 1));
        return (int)(r + (u - more <= 0x7fffffffLL && q <= 0x7fffffffLL ? (unsigned)(u - more) / (unsigned)q : (u - more) / q));
    }
};

// A piece of a CTA's range: windows [i0, i1) of the nw windows of item (w, t, h).
struct SplitPiece {
    int w, t, i0, i1, nw;
    __device__ __forceinline__ bool whole() const { return i0 == 0 && i1 == nw; }
    __device__ __forceinline__ int slot() const { return i0 == 0 ? 1 : 0; }
};
// Walks a range [u, u1) of units; every role of a CTA walks it for itself.
struct SplitWalk {
    long long u, u1, base;  // next unit, end, first unit of sequence w's windows
    int w, nw;              // sequence, its windows per row tile
    // The range of group g, by one whole warp (every lane ends with the same values).  The
    // window counts of up to 256 sequences are loaded at once: one round trip to L2.
    __device__ __forceinline__ void place(const TurnSplit& p, int lane, int g) {
        constexpr int N = 8;
        int v[N];
        long long total = 0;
        for (int w0 = 0; w0 < p.W; w0 += 32 * N) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int x = w0 + 32 * k + lane;
                v[k] = x < p.W ? __ldcg(p.nwin + x) : 0;
            }
#pragma unroll
            for (int k = 0; k < N; ++k) total += v[k];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const SplitRange range(total * p.nt, p);
        u = range.begin(g);
        u1 = range.begin(g + 1);
        base = 0;
        w = p.W;
        nw = 0;
        for (int w0 = 0; w0 < p.W; w0 += 32 * N) {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int x = w0 + 32 * k + lane;
                if (p.W > 32 * N) v[k] = x < p.W ? __ldcg(p.nwin + x) : 0;
                int incl = v[k];
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += up;
                }
                const long long end = base + (long long)incl * p.nt;
                const unsigned hit = __ballot_sync(0xffffffffu, v[k] > 0 && u < end);
                if (hit) {
                    const int src = __ffs(hit) - 1;
                    w = w0 + 32 * k + src;
                    nw = __shfl_sync(0xffffffffu, v[k], src);
                    base = __shfl_sync(0xffffffffu, end, src) - (long long)nw * p.nt;
                    return;
                }
                base = __shfl_sync(0xffffffffu, end, 31);
            }
        }
    }
    __device__ __forceinline__ bool next(const TurnSplit& p, SplitPiece& pc) {
        while (u < u1 && w < p.W) {
            const long long end = base + (long long)nw * p.nt;
            if (u >= end) {
                base = end;
                ++w;
                if (w < p.W) nw = __ldcg(p.nwin + w);
                continue;
            }
            const int local = (int)(u - base);
            pc.w = w;
            pc.nw = nw;
            pc.t = p.nt == 1 ? 0 : local / nw;
            pc.i0 = local - pc.t * nw;
            const long long left = u1 - u;
            pc.i1 = left < nw - pc.i0 ? pc.i0 + (int)left : nw;
            u += pc.i1 - pc.i0;
            return true;
        }
        return false;
    }
};

// The turn and the keys of window i of a sequence: column c of the window is key k0 + c of
// turn f (of the tail where f == F), for c < n and k0 + c >= 0.  Windows are sought in
// increasing order; `start` begins a sequence.
struct SplitWin {
    int f, first, nf, sp, off, k0, n;  // turn, its first window, its windows, seen keys and first position
    bool mixed;                        // some queries see keys of the turn that others do not
    int2 ahead;                        // the next turn's, loaded a turn early
    __device__ __forceinline__ int2 load(const TurnSplit& p, int w, int f_) const {
        return f_ < p.F ? __ldcg(p.span + (size_t)w * p.F + f_) : make_int2(p.tail, 0);
    }
    __device__ __forceinline__ void enter(const TurnSplit& p, int w, int2 x) {
        ahead = load(p, w, f + 1);
        sp = x.x;
        off = x.y & 0x7fffffff;
        mixed = x.y < 0;
        nf = f < p.F ? turn_windows(p, sp, off) : 0x7fffffff - first;
    }
    __device__ __forceinline__ void start(const TurnSplit& p, int w) {
        f = 0, first = 0;
        enter(p, w, load(p, w, 0));
    }
    __device__ __forceinline__ void seek(const TurnSplit& p, int w, int i) {
        while (i >= first + nf) {
            first += nf;
            ++f;
            enter(p, w, ahead);
        }
        k0 = (i - first) * p.kt - (off & (p.align - 1));
        n = min(p.kt, sp - k0);
    }
    // windows from i on that belong to the same turn of the piece
    __device__ __forceinline__ int run(const SplitPiece& pc, int i) const { return min(pc.i1, first + nf) - i; }
};

// A run: consecutive windows of one turn of a piece.  In the warp-specialised kernels one warp
// walks the CTA's range and hands the runs to the others through a ring in shared memory, a few
// ahead, so that none of them keeps the walk's state or waits for its loads.
struct alignas(16) SplitRun {
    int w, t, f, off;    // sequence, row tile (or pass), turn (F: the tail), the turn's first position
    int k0, sp, n, how;  // first key of the first window, seen keys, windows (0: the end), RUN_* bits
};
constexpr int RUN_FIRST = 1, RUN_LAST = 2;   // of its piece
constexpr int RUN_WHOLE = 4, RUN_BEGIN = 8;  // the piece is a whole item; it begins one (SplitPiece::slot)
constexpr int RUN_Q_NEW = 16, RUN_Q_END = 32;  // q rotated for another turn than before; the next run's will be
constexpr int RUN_MIXED = 64;                  // of a turn that is mixed (SplitWin)
constexpr int RUN_RING = 8;

// The walking warp.  passes > 1: every run that many times, t = 0, 1, ..., each with its own q
// (the split then has one row tile).  `full` and `empty` are RUN_RING mbarriers each (one arrival; one per
// consumer).  `tail(w)` is called when the tail of sequence w has been handed out.  false: a wait gave up.
template <class Stop, class Tail>
__device__ __forceinline__ bool split_schedule(const TurnSplit& p, int lane, int g, SplitRun* ring, uint32_t full, uint32_t empty, Stop stopped,
                                               int passes, Tail tail) {
    SplitWalk walk;
    walk.place(p, lane, g);
    SplitPiece pc;
    SplitWin win;
    int n = 0;
    auto push = [&](const SplitRun& r) {
        const int s = n % RUN_RING;
        if (n >= RUN_RING && (stopped() || !__all_sync(0xffffffffu, mbar_wait_lazy(empty + 8 * s, (n / RUN_RING - 1) & 1)))) return false;
        if (lane == 0) {
            ring[s] = r;
            mbar_arrive(full + 8 * s);
        }
        __syncwarp();
        ++n;
        return true;
    };
    while (walk.next(p, pc)) {
        win.start(p, pc.w);
        int turn = -1;
        for (int i = pc.i0; i < pc.i1;) {
            win.seek(p, pc.w, i);
            const int nx = win.run(pc, i), qt = min(win.f, p.F - 1);
            SplitRun r;
            r.w = pc.w, r.t = pc.t, r.f = win.f, r.off = win.off, r.k0 = win.k0, r.sp = win.sp, r.n = nx;
            r.how = (i == pc.i0 ? RUN_FIRST : 0) | (i + nx == pc.i1 ? RUN_LAST : 0) | (pc.whole() ? RUN_WHOLE : 0) | (pc.slot() ? RUN_BEGIN : 0) |
                    (qt != turn ? RUN_Q_NEW : 0) | (i + nx == pc.i1 || qt != p.F - 1 ? RUN_Q_END : 0) | (win.mixed ? RUN_MIXED : 0);
            for (int pass = 0; pass < passes; ++pass) {
                if (passes > 1) r.t = pass, r.how |= RUN_Q_NEW | RUN_Q_END;
                if (!push(r)) return false;
            }
            if (win.f == p.F) tail(pc.w);
            turn = qt;
            i += nx;
        }
    }
    SplitRun end{};
    return push(end);
}

// v, eight 16-bit elements, with zeros for infinities and NaN; true: there was one.
template <class T> __device__ __forceinline__ bool make_finite(uint4& v) {
    constexpr uint32_t top = Elem<T>::dtype == DVATTN_BFLOAT16 ? 0x7f80u : 0x7c00u;
    bool any = false;
    uint32_t* x = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const bool lo = (x[u] & top) == top, hi = (x[u] >> 16 & top) == top;
        if (lo) x[u] &= 0xffff0000u;
        if (hi) x[u] &= 0xffffu;
        any |= lo || hi;
    }
    return any;
}

// A 16-byte chunk (elements e0...) of a row rotated by apply_rotary_pos_emb: o[e] = x[e] c[e] -
// x[e + R/2] s[e], o[e + R/2] = x[e + R/2] c[y] + x[e] s[y] for e < R/2, separate roundings of the
// products and of the sum, one rounding to T.  Queries take y = e (the first half of the cos/sin
// row, as in the paged attention), keys y = e + R/2 (`full`: the whole row; the bits of the
// paged append).  load() issues the chunk's reads, store() computes and writes, so that a
// thread can have several chunks in flight; load_angles() begins another rotation of the same row.
template <class T> struct RotateChunk {
    static constexpr int PER = 16 / (int)sizeof(T);
    uint4 a, b;
    float4 c[PER / 4], s[PER / 4];
    const T* x;
    T* y;
    const float *cos, *sin;
    int e0;
    int back;  // the angle of element e >= R/2 is entry e - back
    __device__ __forceinline__ void load(const T* x_, T* y_, const float* cos_, const float* sin_, int e0_, int R, bool vec) {
        load_row(x_, e0_, R, vec);
        load_angles(y_, cos_, sin_, R, vec);
    }
    __device__ __forceinline__ void load_row(const T* x_, int e0_, int R, bool vec, bool full = false) {
        x = x_, e0 = e0_, back = full ? 0 : R >> 1;
        a = __ldg(reinterpret_cast<const uint4*>(x + e0));
        // vec: rotary halves are whole chunks, cos/sin rows 16-byte aligned
        if (e0 < R && vec) b = __ldg(reinterpret_cast<const uint4*>(x + (e0 < R >> 1 ? e0 + (R >> 1) : e0 - (R >> 1))));
    }
    __device__ __forceinline__ void load_angles(T* y_, const float* cos_, const float* sin_, int R, bool vec) {
        y = y_, cos = cos_, sin = sin_;
        if (e0 < R && vec) {
            const int j = e0 < R >> 1 ? e0 : e0 - back;
#pragma unroll
            for (int u = 0; u < PER / 4; ++u) {
                c[u] = __ldg(reinterpret_cast<const float4*>(cos + j) + u);
                s[u] = __ldg(reinterpret_cast<const float4*>(sin + j) + u);
            }
        }
    }
    __device__ __forceinline__ void store(int R, bool vec) {
        const int half = R >> 1;
        alignas(16) T o[PER];
        *reinterpret_cast<uint4*>(o) = a;
        if (e0 < R && vec) {
            const T* bt = reinterpret_cast<const T*>(&b);
            const float* cf = reinterpret_cast<const float*>(c);
            const float* sf = reinterpret_cast<const float*>(s);
#pragma unroll
            for (int u = 0; u < PER; ++u) {
                const float v = Elem<T>::to_f(bt[u]);
                o[u] = Elem<T>::from_f(__fadd_rn(__fmul_rn(Elem<T>::to_f(o[u]), cf[u]), __fmul_rn(e0 < half ? -v : v, sf[u])));
            }
        } else if (e0 < R) {  // element by element
            for (int u = 0; u < PER && e0 + u < R; ++u) {
                const int e = e0 + u, j = e < half ? e : e - back;
                const float v = Elem<T>::to_f(e < half ? x[e + half] : x[e - half]);
                o[u] = Elem<T>::from_f(__fadd_rn(__fmul_rn(Elem<T>::to_f(x[e]), __ldg(cos + j)), __fmul_rn(e < half ? -v : v, __ldg(sin + j))));
            }
        }
        *reinterpret_cast<uint4*>(y + e0) = *reinterpret_cast<const uint4*>(o);
    }
};
inline bool rotate_vec(int R, const float* cos, const float* sin) {
    return R % 16 == 0 && !((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15);
}

}  // namespace dvb
