// Paged multi-turn decode attention over a cache held in 8 bits (q8.cuh): for token s of sequence w and
// its query head h of KV head k,
//
//   out = sum_l softmax_l(scale * rot_f(q) . (K8_l sk)) (V8_l sv)
//
// over the keys l that (w, s) sees in every turn f, the query rotated for the turn and rounded to its
// type, sk and sv the scales of the key's page and head.  Three launches, each a programmatic dependent of the one before
// it: the rotation of every turn's queries into matrix fragments, the attention, and the merge of the items that more than
// one CTA worked on.
//
// Numerics.  e4m3 is exact in f16, so K and V are widened to f16 in registers and multiplied on
// mma.sync with 32-bit accumulation; the scales never touch them.  q's row is multiplied by a power of
// two that brings its largest element to 2^13 .. 2^14 and written as one f16 value (f16 and bf16 queries:
// exact, but for elements under 2^-27 of the row's largest) or two (f32: hi + lo, within 2^-23 of an
// element), undone in the scores.  With sv = 2^e m (1 <= m < 2), z = log2-score + e is what the running
// maximum r is taken over: P = 2^(z - r + 7), the numerator adds (P m) V8, the denominator P 2^-e, both in
// units of 2^r, so pages of any scales meet in one accumulator.  P m is rounded to f16 (f32: to a hi
// + lo pair) next to V; the denominator adds the unrounded P.  The 7 powers of two keep weights down to
// 2^-21 of the largest at full precision and drop those under 2^-32.  r moves when the maximum has grown by
// more than 6 (P stays below 2^14), so that the accumulators are rarely rescaled.  Values' scales that a row sees have to lie within
// 2^100 of one another: further below the largest, P of a key falls under the least 32-bit number, though P 2^-e would count.
//
// Bound (times of calls replayed from a graph): HBM has a byte per cached element to bring.  128 heads over 4 x 65k to 131k keys
// (843 MB) take 162 us, 80% of the copy bandwidth (a call by itself, on inputs that are not in L2, 180); without any products,
// only windows requested and handed back, it is 151.  The rest is that a byte is also a conversion and products of tensor cores that
// take K and V in 16 bits.  With eight computing warps an SM (190 us) the issue slots were 37% and the tensor cores 28% busy, a warp
// waiting 7 cycles from instruction to instruction: twelve is what the registers hold.  8-bit products would need no conversion, but a
// query would be a sum of e4m3 terms, and one e4m3 mma.sync takes 22 cycles here, the two of f16 that are as deep 20.
// A CTA reads a page's rows of two or four KV heads together (contiguous in HBM) by TMA; a warp works on 16 keys of one
// head.  With 32 keys a warp waits less often but needs more registers, and a range ends further from its share: 32 sequences of
// 64 / 4 heads, bf16, 64.2 us against 57.5; head dim 64, chunks of 5 tokens 82 against 61 (both with two CTAs an SM).
// Rotating the queries in this kernel instead of in a launch of its own cost 4 to 10 us at each turn's start.
#include "decode.cuh"
#include "q8.cuh"
#include "tma_host.cuh"
#include "turns.cuh"

#include <cstdio>
#include <cstdlib>
#include <type_traits>

namespace dvb {

struct Q8Params : TurnSplit {
    // of TurnSplit: F, BS, maxb, cap, NB, kt, nt, align, loc, L, bt
    int first;              // the launch's first pair of all
    int Hq, Hkv, G, S, R, rows;
    int angles;             // entries of a row of cos / sin
    const int* cu;          // packed tokens: where the sequences begin, [nseq + 1]; null: S tokens of each
    int nseq;
    int hc, hs;             // KV heads a CTA reads together, groups of them (hc * hs = Hkv)
    int pairs;              // (sequence, row tile) pairs of the launch, packed tokens: tiles, some of them empty
    int box, box_shift;     // rows of a TMA box (gathered: rows of the stage), its log2
    int bs_shift;           // log2 of the page size, -1: it is no power of two
    long long tokens;       // all sequences' (a turn's stride in loc and cos / sin)
    int stall_tile;         // test hook (DVATTN_TEST_STALL_TILE), -1: off
    float scale_log2;
    void* out;
    float* lse_out;
    float* out_f32;
    const void* q;
    const float* cos;
    const float* sin;
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    // workspace
    int* header;            // [3] error word (kErrorWordOffset)
    const uint8_t* qf;      // [F][pairs][Hkv] {fragments, [rows] factors} of the rotated queries
    const uint8_t* ql;      // [F][pairs] {[rows] keys of the turn that the row sees, the least of them, unused}
    long long* P;           // [pairs + 1] windows in front of a pair (of one head group)
    long long* cstart;      // [CTAs + 1] windows in front of a CTA's
    float* part_o;          // [CTAs][2][hc][rows of a tile][E] sums of weight x value
    float2* part_ml;        // [CTAs][2][hc][rows of a tile] reference m of the weights 2^(score - m + 7), and their sum
};

constexpr int kQ8Warps = 4;
constexpr int kQ8MaxPairs = 2048;  // of a launch: their prefix sums lie in the stages at first
constexpr long long kQ8Fragments = 256LL << 20;  // bytes of rotated queries in the workspace, at most (q8_layout)
// A turn's start (a partial window, its rotated queries, the look-up of its keys) and a piece's end cost about as much as this
// many windows: the split counts them.  96 sequences of 1 to 4 turns, head dim 256: 95.8 us (counted as nothing 107, as eight
// windows 98.2 to 99.4); 32 sequences of two turns 53.4 (four windows 54.5, twelve 54.2).
constexpr int kQ8TurnCost = 6;

// T: the queries' type, E: head dim, MT: 16-row tiles of a KV head's query rows.
template <class T, int E, int MT, bool GATHER> struct Q8Cfg {
    static constexpr int KPW = 16;                      // keys of a warp in a window
    static constexpr int KROWS = kQ8Warps * KPW;        // (key, head) rows of a stage
    static constexpr int TENSOR = KROWS * E;            // bytes of K (or V) in a stage
    static constexpr int NJ = E / 8;                    // 8-column tiles of the output
    static constexpr int ROWS = 16 * MT;
    static constexpr int QT = sizeof(T) == 4 ? 2 : 1, PT = QT;  // f16 values of a query element, of a weight
    static constexpr int KS = E / 16;                           // steps of q . k
    // A head's query fragments: in registers once read, or read for every window, from one of two buffers.
    static constexpr int QFRAG = KS * MT * QT * 512, QHEAD = QFRAG + ROWS * 4;  // ... and the rows' factors
    // Three CTAs of an SM where a warp's sums and one window fit in 128 registers a thread: four computing warps and one that
    // requests all.  Else two (f32 of head dim 256: one) of two warpgroups, registers split between them, with a warp of its own
    // for the queries.  128 heads over 4 x 65k to 131k keys, f16: 170 us against 190; 32 sequences of 64 / 4 heads, bf16, 53.4
    // against 57.5; two row tiles (head dim 64) would spill, 67.9 against 61.5.
    static constexpr bool THREE = QT == 1 && MT == 1 && E <= 128;
    static constexpr bool QREG = !THREE && QFRAG <= 4096;
    static constexpr int QBUFS = QREG ? 1 : 2, HEADS = QREG ? 4 : 2;  // buffers, KV heads of a CTA at most
    static constexpr int LIMS = (ROWS + 4) * 4;                       // what the rows of a tile see, and the least of it
    static constexpr int QBUF = HEADS * QHEAD + LIMS, QBYTES = QBUFS * QBUF;
    static constexpr int CTAS = THREE ? 3 : QBYTES + 4 * TENSOR > 101 * 1024 ? 1 : 2;  // per SM
    static constexpr int LIMIT = CTAS == 3 ? 76800 : CTAS == 2 ? 115712 : 232448;     // shared memory of each
    static constexpr int THREADS = THREE ? 160 : 256;
    // Two CTAs of an SM have 128 registers a thread at their launch; the computing warpgroup takes what the other one
    // gives up.
    static constexpr int REGS = QREG ? 200 : 208, FEW = 2 * 128 - REGS;
    static constexpr int SCALES = GATHER ? KROWS : KROWS / 8;  // of a tensor in a stage: of each row, or of 8 neighbours
    // [warps][ROWS][2] maxima and sums, where several warps share a head (two heads at most: a single
    // query buffer's second half is free)
    static constexpr int ML = QREG ? 0 : kQ8Warps * ROWS * 8;
    static_assert(!QREG || 2 * QHEAD >= kQ8Warps * ROWS * 8, "maxima and sums");
    static constexpr int STAGE = 2 * TENSOR + 2 * SCALES * 4 + 64 + 16;  // tiles, scales, two descriptions (the next window's is written early), barriers
    static constexpr int FIT = (LIMIT - QBYTES - ML - 16 * QBUFS - 12) / STAGE;
    static constexpr int STAGES = FIT > 6 ? 6 : FIT;
    static constexpr size_t OFF_Q = (size_t)STAGES * 2 * TENSOR;
    static constexpr size_t OFF_ML = QREG ? OFF_Q + 2 * QHEAD + LIMS : OFF_Q + QBYTES;
    static constexpr size_t OFF_SC = OFF_Q + QBYTES + ML;               // [STAGES][2][SCALES]
    static constexpr size_t OFF_DESC = OFF_SC + STAGES * 2 * SCALES * 4;
    static constexpr size_t OFF_BAR = OFF_DESC + STAGES * 64;           // full, empty, then q's
    static constexpr size_t OFF_SYNC = OFF_BAR + STAGES * 16 + QBUFS * 16, OFF_FLAG = OFF_SYNC + 8;
    static constexpr size_t SMEM = OFF_FLAG + 4;
    static_assert(STAGES >= 2 && OFF_Q >= (2 * kQ8MaxPairs + 40) * 8, "the prefix sums fit in the stages");
    static_assert(SMEM <= LIMIT && OFF_BAR % 16 == 0, "shared memory");
    static_assert(2 * TENSOR >= 2 * 16 * E * 4, "two heads' rows are combined in a stage");
};

// ---- the windows of a (sequence, row tile) pair ------------------------------------------
struct Q8Tile {
    int table, t, tok0, rows;  // row of the block tables, tile of the sequence, its first token, its rows
    // tokens s0 .. s1 of the sequence (none: s0 > s1)
    __device__ __forceinline__ void tokens(const Q8Params& p, int size, int& s0, int& s1) const {
        s0 = t * size / p.G;
        s1 = t * size < rows ? (min((t + 1) * size, rows) - 1) / p.G : s0 - 1;
    }
};
// Where sequence w of packed tokens begins: as the 16-bit attention reads them, tokens before the first sequence and those
// behind the last one (a sequence `nseq` here) have the first one's table.
__device__ __forceinline__ int packed_start(const Q8Params& p, int w) {
    return w <= 0 ? 0 : w > p.nseq ? (int)p.tokens : min(max(__ldg(p.cu + w), 0), (int)p.tokens);
}
// Packed: sequence w's tiles are those from floor(first row / size) + w on, which leaves room for them all.
// PACKED: a template argument throughout, since the search below in every kernel's start costs a call of the other kind 1 to 3 us.
template <bool PACKED> __device__ __forceinline__ Q8Tile tile_of(const Q8Params& p, int size, int pair) {
    const int x = p.first + pair;
    if constexpr (!PACKED) {
        const int w = x / p.nt;
        return {w, x - w * p.nt, w * p.S, p.rows};
    }
    int w = 0, hi = p.nseq;
    while (w < hi) {
        const int mid = (w + hi + 1) >> 1;
        if ((int)((long long)packed_start(p, mid) * p.G / size) + mid <= x) w = mid; else hi = mid - 1;
    }
    const int tok0 = packed_start(p, w), rows = (packed_start(p, w + 1) - tok0) * p.G;
    return {w < p.nseq ? w : 0, x - ((int)((long long)tok0 * p.G / size) + w), tok0, rows};
}
// of `out`, and of the queries: [token][head] or [sequence][head][token]
template <bool PACKED> __device__ __forceinline__ size_t out_row(const Q8Params& p, int tok0, int head, int s) {
    return PACKED ? (size_t)(tok0 + s) * p.Hq + head : (size_t)tok0 * p.Hq + (size_t)head * p.S + s;
}
// by one thread: {windows, turns that have any}
template <bool PACKED> __device__ __forceinline__ int2 pair_windows(const Q8Params& p, int rows, int pair) {
    const Q8Tile tile = tile_of<PACKED>(p, rows, pair);
    int s0, s1, nw = 0, turns = 0;
    tile.tokens(p, rows, s0, s1);
    if (s0 > s1) return make_int2(0, 0);
    long long off = 0;
    constexpr int AHEAD = 4;  // turns whose lengths and first locations are loaded together
    for (int f0 = 0; f0 < p.F; f0 += AHEAD) {
        int L[AHEAD], at[AHEAD];
#pragma unroll
        for (int x = 0; x < AHEAD; ++x)
            if (f0 + x < p.F) {
                L[x] = __ldg(p.L + f0 + x);
                at[x] = __ldg(p.loc + (f0 + x) * p.tokens + tile.tok0 + s0);
            }
#pragma unroll
        for (int x = 0; x < AHEAD; ++x)
            if (f0 + x < p.F) {
                int sp = turn_seen(L[x], at[x], off, p.cap);
                for (int s = s0 + 1; s <= s1; ++s) sp = max(sp, turn_seen(L[x], __ldg(p.loc + (f0 + x) * p.tokens + tile.tok0 + s), off, p.cap));
                nw += turn_windows(p, sp, sp > 0 ? (int)off : 0);
                turns += sp > 0;
                off += max(L[x], 0);
            }
    }
    return make_int2(nw, turns);
}

// CTA c's units [begin(c), begin(c + 1)): windows and turn starts (kQ8TurnCost each) of all pairs and head groups, evenly split.
struct Q8Split {
    long long q, r;
    int n;
    __device__ __forceinline__ Q8Split(long long total, int ctas) {
        n = total < ctas ? (total > 0 ? (int)total : 1) : ctas;
        q = over(total, n);
        r = total - q * n;
    }
    static __device__ __forceinline__ long long over(long long a, long long b) {  // in 32 bits where both allow
        return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
    }
    __device__ __forceinline__ long long begin(int c) const {
        if (c > n) c = n;
        return c * q + (c < r ? c : r);
    }
};

// What a stage holds: keys [k0, k0 + kt) of a turn of which sp are seen.
struct alignas(16) Q8Stage {
    int k0, sp, how, pad0;  // how: Q8_* bits, -1: the end
    int pair, hg, pad1, pad2;  // what its rows are of
};
static_assert(sizeof(Q8Stage) == 32, "OFF_DESC");
constexpr int Q8_ITEM = 1, Q8_TURN = 2, Q8_LAST = 4, Q8_WHOLE = 8, Q8_BEGIN = 16;

// Window i of turn f of an item; off: the turn's first position, begin: nothing of the item lies in front, before: windows
// in front, of all.
struct alignas(16) Q8Place {
    int pair, hg, f, i;
    long long off, before;
    int begin, pad[3];
};
// Unit `rest` of a pair, by a whole warp, a turn per lane: fills in f, i, off and begin; returns the windows in front.
template <bool PACKED> __device__ __forceinline__ int find_unit(const Q8Params& p, int rows, int lane, int pair, long long rest, Q8Place& at) {
    const Q8Tile tile = tile_of<PACKED>(p, rows, pair);
    int s0, s1, windows = 0;
    tile.tokens(p, rows, s0, s1);
    long long off = 0;
    for (int f0 = 0;; f0 += 32) {
        const bool there = f0 + lane < p.F;
        const int L = there ? __ldg(p.L + f0 + lane) : 0;
        long long sum = max(L, 0);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const long long mine = off + sum - max(L, 0);
        int sp = 0;
        if (there)
            for (int s = s0; s <= s1; ++s) sp = max(sp, turn_seen(L, __ldg(p.loc + (f0 + lane) * p.tokens + tile.tok0 + s), mine, p.cap));
        const int nw = there ? turn_windows(p, sp, sp > 0 ? (int)mine : 0) : 0;
        int upto = nw;
        long long units = nw > 0 ? nw + kQ8TurnCost : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            const long long y = __shfl_up_sync(0xffffffffu, units, o);
            if (lane >= o) upto += x, units += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, units > rest);
        if (past) {
            const int k = __ffs(past) - 1;
            const int own = __shfl_sync(0xffffffffu, nw, k), front = windows + __shfl_sync(0xffffffffu, upto, k) - own;
            const long long in = rest - (__shfl_sync(0xffffffffu, units, k) - own - kQ8TurnCost) - kQ8TurnCost;
            at.f = f0 + k, at.i = in > 0 ? (int)in : 0;
            at.off = __shfl_sync(0xffffffffu, mine, k);
            at.begin = front + at.i == 0;
            return front + at.i;
        }
        rest -= __shfl_sync(0xffffffffu, units, 31);
        windows += __shfl_sync(0xffffffffu, upto, 31);
        off += __shfl_sync(0xffffffffu, sum, 31);
        if (f0 + 32 >= p.F) {  // not reached: rest lies below the pair's units
            at.f = at.i = at.begin = 0, at.off = 0;
            return 0;
        }
    }
}

// Walks the windows of a range by a whole warp; every lane holds the same values.
template <bool PACKED> struct Q8Walk {
    long long rem;
    int pair, hg, f, left;  // left: windows of the turn that are left
    int table;              // the pair's
    int sp, off, k0;        // the turn's seen keys and first position, the next window's first key
    long long off64;
    bool item, turn;  // the next window begins an item's piece, a turn
    bool begin;       // the piece begins its item

    __device__ __forceinline__ void enter(const Q8Params& p, int rows, int lane) {  // turn f
        const int L = __ldg(p.L + f);
        const Q8Tile tile = tile_of<PACKED>(p, rows, pair);
        int s0, s1, v = 0;
        table = tile.table;
        tile.tokens(p, rows, s0, s1);
        for (int s = s0 + lane; s <= s1; s += 32) v = max(v, turn_seen(L, __ldg(p.loc + f * p.tokens + tile.tok0 + s), off64, p.cap));
        sp = __reduce_max_sync(0xffffffffu, v);
        off = sp > 0 ? (int)off64 : 0;
        off64 += max(L, 0);
        left = turn_windows(p, sp, off);
        k0 = -(off & (p.align - 1));
        turn = true;
    }
    // at `at`, for n windows
    __device__ __forceinline__ void start(const Q8Params& p, int rows, int lane, const Q8Place& at, long long n) {
        pair = at.pair, hg = at.hg, rem = n, begin = at.begin != 0, item = true;
        f = at.f, off64 = at.off;
        enter(p, rows, lane);
        k0 += at.i * p.kt;
        left -= at.i;
    }
    __device__ __forceinline__ void skip_turn(const Q8Params& p) {  // its windows that have not been handed out
        const int k = left < rem ? left : (int)rem;
        left -= k, rem -= k, k0 += k * p.kt;
    }
    // To the next window, which begins at key k0; false: none.  `ended`: the windows before end their item.
    __device__ __forceinline__ bool seek(const Q8Params& p, int rows, int lane, bool& ended) {
        ended = false;
        while (left == 0) {
            if (f + 1 < p.F) {
                ++f;
            } else {
                ended = item = begin = true;
                if (rem == 0) return false;
                f = 0, off64 = 0;
                if (++hg == p.hs) {
                    hg = 0;
                    if (++pair >= p.pairs) {
                        rem = 0;
                        return false;
                    }
                }
            }
            enter(p, rows, lane);
        }
        return rem != 0;
    }
    __device__ __forceinline__ int how() const { return (item ? Q8_ITEM : 0) | (turn ? Q8_TURN : 0) | (begin ? Q8_BEGIN : 0); }
    __device__ __forceinline__ void take(const Q8Params& p) {  // past the window
        item = turn = false;
        k0 += p.kt, --left, --rem;
    }
};

// ---- small helpers ------------------------------------------------------------------------
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {  // without an arrival
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {  // when this thread's copies so far have landed
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two 16 x 16 matrices of bytes, rows at the lanes' addresses (0 .. 15 and 16 .. 31): v[0], v[1] get rows 4 (lane % 4) .. + 3 of
// columns lane / 4 and 8 + lane / 4 of the first, v[2], v[3] of the second.
__device__ __forceinline__ void ldsm_b8_t(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(addr)
                 : "memory");
}
template <class T> __device__ __forceinline__ void store_pair(T* dst, float2 x) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(dst) = x;
    else *reinterpret_cast<uint32_t*>(dst) = Elem<T>::pack2(x.x, x.y);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { return Elem<__half>::pack2(a, b); }

// v = 2^e m of a scale (file comment), e at least -60; what is not finite or not positive comes out in m.
struct Scale {
    float e, m, inv;  // inv = 2^-e
    __device__ __forceinline__ Scale(float v) {
        const int b = __float_as_int(v), x = b & 0x7f800000;
        const bool low = b < (67 << 23), odd = x == 0x7f800000;
        e = low ? -60.f : __int_as_float((b >> 23) + 0x4b000000) - (8388608.f + 127.f);
        m = low ? v * 0x1p60f : odd ? v : __int_as_float((b & 0x7fffff) | 0x3f800000);
        inv = low ? 0x1p60f : odd ? 0x1p-128f : __int_as_float(0x7f000000 - x);
    }
};
__device__ const float kOne = 1.f;

// ---- the rotation ----------------------------------------------------------------------------
// Block (f, pair, h): the tile's query rows of KV head h rotated for turn f, scaled and split into the fragments that
// the attention kernel reads (below), E / 8 lanes per row.  It runs while the attention kernel finds its split and requests
// its first windows.  By the attention kernel's own warps, a turn took 4 to 10 us, in rounds of loads that few
// registers allow.
template <class T, int E, int MT, bool PACKED> __global__ void __launch_bounds__(128) rotate_q8_kernel(const __grid_constant__ Q8Params p, uint8_t* qf, uint8_t* ql) {
    using C = Q8Cfg<T, E, MT, false>;
    constexpr int ROWS = C::ROWS, KS = C::KS, LPR = E / 8, STEP = 128 / LPR;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int h = blockIdx.x % p.Hkv, fp = blockIdx.x / p.Hkv, f = fp / p.pairs, pair = fp - f * p.pairs;
    const int tid = threadIdx.x;
    const Q8Tile tile = tile_of<PACKED>(p, ROWS, pair);
    const int t = tile.t;
    long long off = 0;
    for (int x = 0; x < f; ++x) off += max(__ldg(p.L + x), 0);
    const int L = __ldg(p.L + f);
    int s0, s1, sp = 0;
    tile.tokens(p, ROWS, s0, s1);
    if (s0 > s1) return;
    const int* loc = p.loc + f * p.tokens + tile.tok0;
    const bool vec = p.R % 16 == 0 && !((reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin)) & 15);
    const int ch = tid % LPR;
    float v[ROWS / STEP][8];
#pragma unroll
    for (int i = 0; i < ROWS / STEP; ++i) {
        const int row = t * ROWS + i * STEP + tid / LPR;
#pragma unroll
        for (int u = 0; u < 8; ++u) v[i][u] = 0.f;
        if (row < tile.rows) {
            const int s = row / p.G;
            const size_t angle = (f * p.tokens + tile.tok0 + s) * p.angles;
            rotated8<T, false>(static_cast<const T*>(p.q) + out_row<PACKED>(p, tile.tok0, h * p.G + row - s * p.G, s) * E, p.cos + angle, p.sin + angle, 8 * ch, p.R, vec,
                               v[i]);
        }
    }
    for (int s = s0; s <= s1; ++s) sp = max(sp, turn_seen(L, __ldg(loc + s), off, p.cap));
    if (sp == 0) return;  // nobody reads the turn
    if (h == 0 && tid < 32) {
        const int row = t * ROWS + tid, see = tid < ROWS && row < tile.rows ? turn_seen(L, __ldg(loc + row / p.G), off, p.cap) : sp;
        int* dst = reinterpret_cast<int*>(ql + (size_t)fp * C::LIMS);
        if (tid < ROWS) dst[tid] = see;
        const int least = __reduce_min_sync(0xffffffffu, see);
        if (tid == 0) dst[ROWS] = least;
    }
    uint8_t* head = qf + (size_t)blockIdx.x * C::QHEAD;
#pragma unroll
    for (int i = 0; i < ROWS / STEP; ++i) {
        const int i16 = i * STEP + tid / LPR;
        float top = 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) top = fmaxf(top, fabsf(v[i][u]));
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int shift = min(140 - (__float_as_int(top) >> 23), 126);
        const float mul = __int_as_float((127 + shift) << 23);
        if (ch == 0) reinterpret_cast<float*>(head + C::QFRAG)[i16] = p.scale_log2 * __int_as_float((127 - shift) << 23);
        // chunk t + 4j of row n + 8 half of tile mt, lane (n, t)'s: step 4j + u, a[half] = elements 4u, 4u + 1, a[2 + half] the next two
        const int c16 = ch >> 1;
        uint8_t* dst = head + ((i16 >> 4) * C::QT * KS + 4 * (c16 >> 2) + 2 * (ch & 1)) * 512 + ((i16 & 7) * 4 + (c16 & 3)) * 16 + (i16 >> 3 & 1) * 4;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float x[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) x[y] = v[i][u * 4 + y] * mul;
#pragma unroll
            for (int term = 0; term < C::QT; ++term) {
                const uint32_t lo = pack_f16(x[0], x[1]), hi = pack_f16(x[2], x[3]);
                *reinterpret_cast<uint32_t*>(dst + (term * KS + u) * 512) = lo;
                *reinterpret_cast<uint32_t*>(dst + (term * KS + u) * 512 + 8) = hi;
                const __half2 a = *reinterpret_cast<const __half2*>(&lo), b = *reinterpret_cast<const __half2*>(&hi);
                x[0] -= __low2float(a), x[1] -= __high2float(a), x[2] -= __low2float(b), x[3] -= __high2float(b);
            }
        }
    }
}

// Natural logarithm of weights 2^(score - m + 7) that add up to `sum`; m = -inf: none are seen, or their sum is NaN.
__device__ __forceinline__ float log_sum(float m, float sum) {
    return sum == 0.f ? neg_inf() : ((m == neg_inf() ? 0.f : m - 7.f) + log2f(sum)) * kLn2;
}

// ---- the attention kernel ---------------------------------------------------------------------
// Warps 0 .. 3 compute, warp 4 requests the windows and, with 160 threads, the rotated queries (else warp 5).  Warp w works on head w % hc of the group and keys
// [KPW (w / hc), + KPW) of the window; thread (n, t) = (lane / 4, lane % 4).
//
// Fragments.  The order of the elements in q . k and of the keys in P V is free as long as both operands
// share it:
// * K comes in 16-byte words: thread (n, t) takes chunks t + 4i of the rows of its columns n and widens each 32-bit word to a
//   fragment.  (8-bit products would take K as it is, at the file comment's cost.)
// * V comes by transposing 8-bit matrix loads: thread (n, t) gets, of column n, the keys of rows 4t .. 4t + 3, and
//   widens them in pairs to a fragment.  So the scores that a thread holds have to be those of these four keys: of 16 keys,
//   key(t, j) = 8 (t / 2) + 2 (t % 2) + j / 2 + 4 (j % 2) for tile j / 2, column 2t + j % 2.  Neighbouring columns lie four rows
//   apart and eight rows in a row differ, which the 128-byte swizzle puts in different banks, and a thread's
//   four keys lie in 8 neighbouring rows: one page, one scale.
template <class T, int E, int MT, bool GATHER, bool PACKED>
__global__ void __launch_bounds__((Q8Cfg<T, E, MT, GATHER>::THREADS), (Q8Cfg<T, E, MT, GATHER>::CTAS))
    decode_q8_kernel(const __grid_constant__ Q8Params p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
    using C = Q8Cfg<T, E, MT, GATHER>;
    constexpr int QT = C::QT, PT = C::PT;
    constexpr int KPW = C::KPW, KS = C::KS, NJ = C::NJ, STAGES = C::STAGES, ROWS = C::ROWS;
    constexpr int RB = E < 128 ? E : 128;  // bytes of a swizzled row
    constexpr int NP = E / RB;             // panels
    constexpr int NTH = C::THREADS;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t s0 = smem_u32(smem);
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const uint32_t bar_full = s0 + (uint32_t)C::OFF_BAR, bar_empty = bar_full + STAGES * 8, bar_q = bar_empty + STAGES * 8;
    volatile int* stop = reinterpret_cast<volatile int*>(smem + C::OFF_FLAG);
    Q8Stage* desc = reinterpret_cast<Q8Stage*>(smem + C::OFF_DESC);
    if (tid == 0) {
        for (int st = 0; st < STAGES; ++st) {
            mbar_init(bar_full + st * 8, 33);  // the description and the loading lanes' copies
            mbar_init(bar_empty + st * 8, kQ8Warps);
        }
        for (int x = 0; x < C::QBUFS; ++x) {
            mbar_init(bar_q + x * 16, 1);
            mbar_init(bar_q + x * 16 + 8, kQ8Warps);  // free again
        }
        mbar_init(s0 + (uint32_t)C::OFF_SYNC, kQ8Warps);
        *stop = 0;
        fence_mbar_init();
    }
    // A programmatic dependent of the rotation, whose blocks let this grid begin once whatever is before them has ended: the
    // call's inputs and outputs are free.  What the rotation writes is waited for where it is read.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int c = blockIdx.x;
    const bool aligned = (s0 & 1023) == 0;  // as the swizzle needs the stages
    // cleared once per call: a bounded wait that gives up sets its bit long after
    if (c == 0 && tid == 0 && (p.first == 0 || !aligned)) p.header[3] = aligned ? 0 : 4;
    if (!aligned) return;
    // ---- the split: every CTA adds up the windows and units of all pairs and finds its own range ----
    long long* sP = reinterpret_cast<long long*>(smem);  // [pairs + 1] windows in front of a pair, in the stages
    long long* sU = sP + p.pairs + 1;                    // [pairs + 1] units
    long long* scratch = sU + p.pairs + 1;
    long long carry = 0, carry_u = 0;
    for (int base = 0; base < p.pairs; base += NTH) {
        const int pair = base + tid;
        const int2 own = pair < p.pairs ? pair_windows<PACKED>(p, ROWS, pair) : make_int2(0, 0);
        const long long own_u = own.x + (long long)kQ8TurnCost * own.y;
        long long x = own.x, u = own_u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o), yu = __shfl_up_sync(0xffffffffu, u, o);
            if (lane >= o) x += y, u += yu;
        }
        if (lane == 31) scratch[wid] = x, scratch[8 + wid] = u;
        __syncthreads();
        long long before = carry, before_u = carry_u;
        for (int y = 0; y < NTH / 32; ++y) {
            if (y < wid) before += scratch[y], before_u += scratch[8 + y];
            carry += scratch[y], carry_u += scratch[8 + y];
        }
        if (pair < p.pairs) sP[pair] = before + x - own.x, sU[pair] = before_u + u - own_u;
        __syncthreads();
    }
    if (tid == 0) sP[p.pairs] = carry, sU[p.pairs] = carry_u;
    __syncthreads();
    for (int i = c * NTH + tid; i <= p.pairs; i += gridDim.x * NTH) p.P[i] = sP[i];  // for the merge
    Q8Place* place = reinterpret_cast<Q8Place*>(scratch);                            // of the range's two ends
    if (wid < 2) {
        const Q8Split split(carry_u * p.hs, gridDim.x);
        const long long u = split.begin(c + wid);
        Q8Place at{};
        at.pair = p.pairs, at.before = carry * p.hs;
        if (u < carry_u * p.hs) {
            int pair = 0, hi = p.pairs - 1;
            while (pair < hi) {  // the last pair that begins at or before u; those without windows begin with the next
                const int mid = (pair + hi + 1) >> 1;
                if (sU[mid] * p.hs <= u) pair = mid; else hi = mid - 1;
            }
            const long long local = u - sU[pair] * p.hs, units = sU[pair + 1] - sU[pair];
            at.pair = pair, at.hg = (int)Q8Split::over(local, units);
            at.before = sP[pair] * p.hs + at.hg * (sP[pair + 1] - sP[pair]);
            at.before += find_unit<PACKED>(p, ROWS, lane, pair, local - at.hg * units, at);
        }
        if (lane == 0) {
            place[wid] = at;
            if (wid == 0) p.cstart[c] = at.before;
            else if (c == (int)gridDim.x - 1) p.cstart[c + 1] = at.before;
        }
    }
    fence_proxy_async_smem();  // TMA writes where the sums lay
    __syncthreads();
    const Q8Place from = place[0];
    const long long count = place[1].before - from.before;
    __syncthreads();
    if (count <= 0) return;

    if (wid >= kQ8Warps) {
        if constexpr (C::CTAS == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::FEW));
        if (wid > kQ8Warps + 1) return;
        // Requests the fragments of turn f of head group hg of a pair, the n-th of this CTA; false: a wait gave up.
        auto request_q = [&](int n, int f, int pair, int hg) {
            if (n == 0) {
                asm volatile("griddepcontrol.wait;" ::: "memory");
                asm volatile("fence.proxy.async;" ::: "memory");  // written with ordinary stores, read by bulk copies
            }
            const int buf = n % C::QBUFS;
            if (n >= C::QBUFS && (__any_sync(0xffffffffu, *stop != 0) || !__all_sync(0xffffffffu, mbar_wait(bar_q + buf * 16 + 8, (n / C::QBUFS - 1) & 1)))) return false;
            if (lane == 0) {
                const uint32_t dst = s0 + (uint32_t)(C::OFF_Q + (size_t)buf * C::QBUF);
                const size_t at = (size_t)f * p.pairs + pair;
                mbar_expect_tx(bar_q + buf * 16, (uint32_t)(p.hc * C::QHEAD + C::LIMS));
                bulk_load(dst, p.qf + (at * p.Hkv + (size_t)hg * p.hc) * C::QHEAD, p.hc * C::QHEAD, bar_q + buf * 16);
                bulk_load(dst + (uint32_t)(p.hc * C::QHEAD), p.ql + at * C::LIMS, C::LIMS, bar_q + buf * 16);
            }
            __syncwarp();
            return true;
        };
        if (!C::THREE && wid == kQ8Warps + 1) {  // a warp of its own for them
            Q8Walk<PACKED> walk;
            walk.start(p, ROWS, lane, from, count);
            bool ended;
            for (int n = 0; walk.seek(p, ROWS, lane, ended); ++n) {
                if (!request_q(n, walk.f, walk.pair, walk.hg)) {
                    if (lane == 0) {
                        *stop = 1;
                        atomicOr(p.header + 3, 1);
                    }
                    break;
                }
                walk.skip_turn(p);
            }
            return;
        }
        // ======================= the requesting warp =======================
        // A window ahead of its requests: where its pages are has been looked up by then.  What does not change from window to
        // window is worked out once: a window's turn came to 1.7 us otherwise, as long as HBM takes to bring it.
        const int boxes = p.kt >> p.box_shift, hc_shift = p.hc >> 1;  // 1, 2, 4
        if (lane == 0 && !GATHER) {
            prefetch_tmap(&mk);
            prefetch_tmap(&mv);
        }
        const uint32_t box_at = (uint32_t)(lane * p.box * p.hc * E);  // of this lane's box in a tile
        // this lane's scale (pages that are whole boxes): of head y % hc, keys 8 (y / hc) .. + 7 of K's or V's tile
        const int per = p.kt / 8 * p.hc, sy = lane < per ? lane : lane - per;
        const bool scales = lane < 2 * per;
        const float* sbase = (lane < per ? p.ks : p.vs) + (sy & (p.hc - 1));
        const uint32_t sat = s0 + (uint32_t)(C::OFF_SC + 4 * (sy + (lane < per ? 0 : C::SCALES)));
        const int sbox = (sy >> hc_shift) * 8 >> p.box_shift & 31;
        Q8Walk<PACKED> walk;
        walk.start(p, ROWS, lane, from, count);
        // of the next window: lane's box, or (gathered) keys lane + 32 x: its page (-1: none) and row there
        constexpr int NX = GATHER ? 4 : 1;
        int page[NX], inpage[NX], how = 0, hg = 0;
        bool have, ended;
        auto find = [&](int i) {
            have = walk.seek(p, ROWS, lane, ended);
            if (!have) return;
            const int n = GATHER ? p.kt : boxes, step = GATHER ? 1 : p.box;
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                const int k = lane + 32 * x, l = walk.k0 + k * step, pos = walk.off + l;
                page[x] = -1;
                if (k < n && l + step > 0 && l < walk.sp) {
                    const int at = p.bs_shift >= 0 ? pos >> p.bs_shift : pos / p.BS;
                    inpage[x] = pos - at * p.BS;
                    page[x] = __ldg(p.bt + (size_t)walk.table * p.maxb + at);
                }
            }
            how = walk.how();
            hg = walk.hg;
            if (lane == 0) {
                Q8Stage& d = desc[i % (2 * STAGES)];
                d.k0 = walk.k0, d.sp = walk.sp;
                d.pair = walk.pair, d.hg = hg;
            }
            walk.take(p);
        };
        find(0);
        bool ok = true;
        int i = 0;
        [[maybe_unused]] int turns = 0;
        for (;; ++i) {
            const int st = i % STAGES;
            const uint32_t full = bar_full + st * 8;
            if (i >= STAGES && (__any_sync(0xffffffffu, *stop != 0) || !__all_sync(0xffffffffu, mbar_wait(bar_empty + st * 8, (i / STAGES - 1) & 1)))) {
                ok = false;
                break;
            }
            if (!have) {
                if (lane == 0) {
                    desc[i % (2 * STAGES)].how = -1;
                    mbar_arrive(full);
                }
                mbar_arrive(full);
                break;
            }
            int pg[NX], row[NX], what = how;
            const int heads = hg * p.hc;  // the first head
            if constexpr (!GATHER) {
                if (i != p.stall_tile || c != 0) {  // test hook: that stage is never filled
                    if (lane == 0) mbar_expect(full, 2u * C::TENSOR);
                    __syncwarp();
                    const int b = page[0] < p.NB ? page[0] : -1;
                    if (lane < boxes) {
                        const int z = b >= 0 ? b * p.BS + inpage[0] : -2 * p.box;  // rows outside: zeros
                        const uint32_t dk = s0 + (uint32_t)(st * 2 * C::TENSOR) + box_at;
                        tma_load_4d(dk, &mk, 0, z, 0, heads, full);
                        tma_load_4d(dk + C::TENSOR, &mv, 0, z, 0, heads, full);
                    }
                    const int sb = __shfl_sync(0xffffffffu, b, sbox);
                    if (scales) cp_async4(sat + (uint32_t)(st * 2 * C::SCALES * 4), sb >= 0 ? sbase + (size_t)sb * p.Hkv + heads : &kOne);
                }
            } else {
#pragma unroll
                for (int x = 0; x < NX; ++x) pg[x] = page[x] < p.NB ? page[x] : -1, row[x] = inpage[x];
            }
            if (C::THREE && (what & Q8_TURN) && !request_q(turns++, walk.f, walk.pair, hg)) {
                ok = false;
                ++i;
                break;
            }
            find(i + 1);
            // the item's piece ends here where the next window begins another or there is none
            if (!have || (how & Q8_ITEM)) what |= Q8_LAST | (ended && (what & Q8_BEGIN) ? Q8_WHOLE : 0);
            if (i == p.stall_tile && c == 0) continue;
            if (lane == 0) {
                desc[i % (2 * STAGES)].how = what;
                mbar_arrive(full);  // the description is there
            }
            if constexpr (GATHER) {
                // 16-byte chunk ch of row (head, key): [head][panel][KT keys][RB bytes], swizzled as TMA writes it
                const uint32_t dk = s0 + (uint32_t)(st * 2 * C::TENSOR), dv = dk + C::TENSOR;
                const uint32_t sc = s0 + (uint32_t)C::OFF_SC + (uint32_t)(st * 2 * C::SCALES * 4);
                auto of_key = [&](const int (&v)[NX], int key) {
                    const int v0 = __shfl_sync(0xffffffffu, v[0], key & 31), v1 = __shfl_sync(0xffffffffu, v[1], key & 31);
                    const int v2 = __shfl_sync(0xffffffffu, v[2], key & 31), v3 = __shfl_sync(0xffffffffu, v[3], key & 31);
                    return key < 32 ? v0 : key < 64 ? v1 : key < 96 ? v2 : v3;
                };
                constexpr int CH = E / 16;
                for (int x = lane; x < C::KROWS * CH; x += 32) {
                    const int r = x / CH, ch = x % CH, hh = r / p.kt, key = r - hh * p.kt;
                    const int b = of_key(pg, key), in = of_key(row, key);
                    const size_t at = b >= 0 ? (((size_t)b * p.BS + in) * p.Hkv + heads + hh) * E + ch * 16 : 0;
                    const uint32_t panel = (uint32_t)((hh * NP + ch / (RB / 16)) * p.kt + key) * RB;
                    const uint32_t to = panel + (uint32_t)((RB == 128 ? (ch & 7) ^ (key & 7) : ch ^ (key >> 1 & 3)) << 4);
                    cp_async16_zfill(dk + to, p.k + at, b >= 0 ? 16 : 0);
                    cp_async16_zfill(dv + to, p.v + at, b >= 0 ? 16 : 0);
                }
                for (int x = lane; x < C::KROWS; x += 32) {  // scales, [key][head]
                    const int b = of_key(pg, x >> hc_shift);
                    const size_t at = (size_t)b * p.Hkv + heads + (x & (p.hc - 1));
                    cp_async4(sc + 4 * x, b >= 0 ? p.ks + at : &kOne);
                    cp_async4(sc + 4 * (x + C::SCALES), b >= 0 ? p.vs + at : &kOne);
                }
            }
            cp_async_arrive(full);
        }
        if (!ok) {
            if (lane == 0) {
                *stop = 1;
                atomicOr(p.header + 3, 1);
            }
            cp_async_commit();
            cp_async_wait<0>();
            for (int j = max(0, i - STAGES); j < i; ++j)  // what was requested lands first (bounded)
                if (j != p.stall_tile || c != 0) mbar_wait(bar_full + (j % STAGES) * 8, (j / STAGES) & 1);
        }
        return;
    }

    // =========================== computing warps ===========================
    if constexpr (C::CTAS == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS));
    const int n = lane >> 2, t = lane & 3;
    const int hh = wid % p.hc, grp = wid / p.hc, wph = kQ8Warps / p.hc;  // head of the group, warps per head
    const int kw = grp * KPW;                                            // first key of the window
    // 8 neighbouring keys x: their rows' place in a stage's K (V), a panel further: + panel
    auto rows8 = [&](int x) {
        const int key = kw + 8 * x, b = key >> p.box_shift;
        return (uint32_t)(((b * p.hc + hh) * NP * p.box + (key & (p.box - 1))) * RB);
    };
    auto swizzle = [](int row) { return (uint32_t)(RB == 128 ? row & 7 : row >> 1 & 3); };  // of a row's 16-byte chunks
    const uint32_t panel = (uint32_t)(p.box * RB);
    constexpr int NT = KPW / 8;              // 8-key tiles
    uint32_t kofs[2][E < 128 ? 1 : 2];       // K rows of column n, by tile and chunk t or t + 4
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int row = (n >> 1 & 1) * 2 + x + 4 * (n & 1);
#pragma unroll
        for (int y = 0; y < (E < 128 ? 1 : 2); ++y) kofs[x][y] = rows8(n >> 2) + (uint32_t)(row * RB) + (((t + 4 * y) ^ swizzle(row)) << 4);
    }
    // V rows of a matrix load: lanes 0 .. 15 the keys' 16 bytes of a block of columns, 16 .. 31 of the next one
    uint32_t vrow;
    {
        const int t4 = lane >> 2 & 3, j = lane & 3, key = (t4 >> 1) * 8 + (t4 & 1) * 2 + (j >> 1) + 4 * (j & 1), half = lane >> 4;
        vrow = rows8(key >> 3) + (uint32_t)((key & 7) * RB) + ((swizzle(key & 7) ^ (uint32_t)half) << 4);
    }
    const int mykey = (t >> 1) * 8 + (t & 1) * 2;  // key(t, 0)
    uint32_t sQ = 0;  // this lane's fragments of the turn's buffer
    int nq = 0;       // turns so far
    float* sML = reinterpret_cast<float*>(smem + C::OFF_ML);

    uint32_t qf[C::QREG ? MT * QT * KS : 1][4];
    float fr[MT][2];   // log2(e) * scale / (the row's power of two)
    int lim[MT][2];    // keys of the turn that the row sees
    int least = 0;     // that every row of the warp sees
    float o[MT][NJ][4], r[MT][2];
    uint64_t l[MT][2];  // two sums each

    // The next turn's fragments and row values; false: a wait gave up.
    auto take_q = [&] {
        const int buf = nq % C::QBUFS;
        if (!__all_sync(0xffffffffu, mbar_wait(bar_q + buf * 16, (nq / C::QBUFS) & 1))) return false;
        const uint32_t base = s0 + (uint32_t)(C::OFF_Q + (size_t)buf * C::QBUF), head = base + (uint32_t)(hh * C::QHEAD);
        const uint32_t limits = base + (uint32_t)(p.hc * C::QHEAD);
        sQ = head + lane * 16;
        if constexpr (C::QREG) {
#pragma unroll
            for (int x = 0; x < MT * QT * KS; ++x) {
                const uint4 v = lds128(sQ + x * 512);
                qf[x][0] = v.x, qf[x][1] = v.y, qf[x][2] = v.z, qf[x][3] = v.w;
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                fr[mt][y] = lds_f32(head + C::QFRAG + 4 * (mt * 16 + y * 8 + n));
                lim[mt][y] = __float_as_int(lds_f32(limits + 4 * (mt * 16 + y * 8 + n)));
            }
        least = __float_as_int(lds_f32(limits + 4 * ROWS));
        // the buffer that is free now: this one, or (fragments are read for every window) the one before
        __syncwarp();
        if (lane == 0 && (C::QREG || nq > 0)) mbar_arrive(bar_q + (C::QREG ? buf : buf ^ 1) * 16 + 8);
        ++nq;
        return true;
    };

    // One window's keys [first, first + KPW) of this warp.  EDGE: some row does not see them all.
    auto window = [&](auto edge, int sp, int first, uint32_t kb, uint32_t sc) {
        constexpr bool EDGE = decltype(edge)::value;
        const uint32_t vb = kb + C::TENSOR;
        auto key_of = [&](int x, int y) { return mykey + x + 4 * y; };  // of tile x, this thread's column y
        auto sees = [&](int x, int y, int mt, int half) {
            const int key = first + key_of(x, y);
            return key >= 0 && key < lim[mt][half];
        };
        // ---- scores ----
        float z[MT][NT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int x = 0; x < NT; ++x) z[mt][x][0] = z[mt][x][1] = z[mt][x][2] = z[mt][x][3] = 0.f;
#pragma unroll
        for (int ci = 0; ci < E / 64; ++ci) {
            // f32: the sum of 64 elements by itself, added with one rounding (a tensor core's sum cuts at every step)
            [[maybe_unused]] float part[NT][4] = {};
            uint4 kf[NT];
#pragma unroll
            for (int x = 0; x < NT; ++x) kf[x] = lds128(kb + (ci >> 1) * panel + kofs[x][E < 128 ? 0 : ci & 1]);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int ks = 4 * ci + u;
                uint32_t a[MT * QT][4];
#pragma unroll
                for (int y = 0; y < MT * QT; ++y) {
                    if constexpr (C::QREG) {
#pragma unroll
                        for (int v = 0; v < 4; ++v) a[y][v] = qf[y * KS + ks][v];
                    } else {
                        const uint4 v = lds128(sQ + (uint32_t)((y * KS + ks) * 512));
                        a[y][0] = v.x, a[y][1] = v.y, a[y][2] = v.z, a[y][3] = v.w;
                    }
                }
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    const uint32_t word = u == 0 ? kf[x].x : u == 1 ? kf[x].y : u == 2 ? kf[x].z : kf[x].w;
                    const uint32_t b0 = e4m3x2_to_f16x2(word), b1 = e4m3x2_hi_to_f16x2(word);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int term = QT - 1; term >= 0; --term) mma_f16(QT > 1 && term == 0 ? part[x] : z[mt][x], a[mt * QT + term], b0, b1);
                }
            }
            if constexpr (QT > 1) {
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int y = 0; y < 4; ++y) z[0][x][y] += part[x][y];
            }
        }
        constexpr int TJ = 4, AHEAD = 2;  // output tiles of a load of V; loads under way
        uint32_t vals[AHEAD][4];
        auto load_v = [&](int j0) {
            const int cb = j0 >> 1;  // 16-column block
            ldsm_b8_t(((vb + (cb >> 3) * panel) + vrow) ^ (uint32_t)((cb & 7) << 4), vals[j0 / TJ % AHEAD]);
        };
#pragma unroll
        for (int j0 = 0; j0 < AHEAD * TJ && j0 < NJ; j0 += TJ) load_v(j0);
        // ---- weights ----
        // scales of this thread's keys: their one page's, or each key's own
        constexpr int NS = GATHER ? 4 : 1;
        float vscale[NS];
#pragma unroll
        for (int k = 0; k < NS; ++k) {  // key(t, k): tile k / 2, column k % 2
            const int at = (GATHER ? kw + key_of(k >> 1, k & 1) : (kw >> 3) + (t >> 1)) * p.hc + hh;
            const float ks = lds_f32(sc + 4 * at);
            vscale[k] = lds_f32(sc + 4 * (at + C::SCALES));
            const float e = Scale(vscale[k]).e;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float f = ks * fr[mt][half];
                    if constexpr (GATHER) {
                        float& x = z[mt][k >> 1][2 * half + (k & 1)];
                        x = fmaf(x, f, e);
                    } else {
#pragma unroll
                        for (int x = 0; x < NT; ++x) {
                            float* y = z[mt][x] + 2 * half;
                            u2f(ffma2(f2u(y[0], y[1]), f2u(f, f), f2u(e, e)), y[0], y[1]);
                        }
                    }
                }
        }
        if constexpr (EDGE) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        if (!sees(x, y & 1, mt, y >> 1)) z[mt][x][y] = neg_inf();
        }
        bool moves = false;
        float top[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float m = fmax3(fmaxf(z[mt][0][2 * y], z[mt][0][2 * y + 1]), z[mt][1][2 * y], z[mt][1][2 * y + 1]);
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                top[mt][y] = m;
                moves |= m > r[mt][y] + 6.f;
            }
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const bool up = top[mt][y] > r[mt][y] + 6.f;
                    const float alpha = up ? fast_exp2(r[mt][y] - top[mt][y]) : 1.f;
                    if (up) r[mt][y] = top[mt][y];
                    l[mt][y] = fmul2(l[mt][y], f2u(alpha, alpha));
#pragma unroll
                    for (int j = 0; j < NJ; ++j) o[mt][j][2 * y] *= alpha, o[mt][j][2 * y + 1] *= alpha;
                }
        }
        uint32_t pa[MT][PT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float ref = r[mt][half] == neg_inf() ? 0.f : r[mt][half] - 7.f;
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    float w[2];
                    u2f(fadd2(f2u(z[mt][x][2 * half], z[mt][x][2 * half + 1]), f2u(-ref, -ref)), w[0], w[1]);
                    w[0] = fast_exp2(w[0]), w[1] = fast_exp2(w[1]);
                    const Scale s0(vscale[GATHER ? 2 * x : 0]), s1(vscale[GATHER ? 2 * x + 1 : 0]);
                    if constexpr (EDGE) {  // what a masked key's scales are does not matter
                        float a, b;
                        u2f(l[mt][half], a, b);
                        const bool see0 = sees(x, 0, mt, half), see1 = sees(x, 1, mt, half);
                        if (see0) a = fmaf(w[0], s0.inv, a);
                        if (see1) b = fmaf(w[1], s1.inv, b);
                        l[mt][half] = f2u(a, b);
                        w[0] = see0 ? w[0] * s0.m : 0.f;
                        w[1] = see1 ? w[1] * s1.m : 0.f;
                    } else {
                        l[mt][half] = ffma2(f2u(w[0], w[1]), f2u(s0.inv, s1.inv), l[mt][half]);
                        u2f(fmul2(f2u(w[0], w[1]), f2u(s0.m, s1.m)), w[0], w[1]);
                    }
#pragma unroll
                    for (int term = 0; term < PT; ++term) {
                        const uint32_t a = pack_f16(w[0], w[1]);
                        pa[mt][term][x * 2 + half] = a;
                        if constexpr (PT > 1) {
                            const __half2 h2 = *reinterpret_cast<const __half2*>(&a);
                            w[0] -= __low2float(h2), w[1] -= __high2float(h2);
                        }
                    }
                }
            }
        // ---- P V, a matrix load (4 output tiles) at a time, AHEAD of them under way ----
        [[maybe_unused]] uint32_t seen = 0u;  // the bytes of this thread's keys that anybody sees
        if constexpr (EDGE) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int key = first + key_of(k >> 1, k & 1);
                if (key >= 0 && key < sp) seen |= 0xffu << (8 * k);
            }
        }
#pragma unroll
        for (int j0 = 0; j0 < NJ; j0 += TJ) {
            uint32_t(&v)[4] = vals[j0 / TJ % AHEAD];
            if constexpr (EDGE) {
                // keys that nobody sees: zeros.  A NaN in the value of a key that some rows see and others do not (0 * NaN
                // is NaN) becomes a zero here and is added to the rows that see it.
                bool odd = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] &= seen;
                    odd |= e4m3_nan(v[i]) != 0;
                }
                if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        uint32_t ind[4];  // 1 where the row sees the key
#pragma unroll
                        for (int x = 0; x < NT; ++x)
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                ind[x * 2 + half] = (sees(x, 0, mt, half) ? 0x3c00u : 0u) | (sees(x, 1, mt, half) ? 0x3c000000u : 0u);
#pragma unroll
                        for (int j = 0; j < TJ; ++j) {
                            float cnt[4] = {0.f, 0.f, 0.f, 0.f};
                            const uint32_t nan = e4m3_nan(v[j]);
                            mma_f16(cnt, ind, (nan & 0x80u ? 0x3c00u : 0u) | (nan & 0x8000u ? 0x3c000000u : 0u),
                                    (nan & 0x800000u ? 0x3c00u : 0u) | (nan & 0x80000000u ? 0x3c000000u : 0u));
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                if (cnt[y] > 0.f) o[mt][j0 + j][y] = __int_as_float(0x7fc00000);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = clear_bytes(v[i], e4m3_nan(v[i]));
                }
            }
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                const uint32_t b0 = e4m3x2_to_f16x2(v[j]), b1 = e4m3x2_hi_to_f16x2(v[j]);
                if constexpr (PT > 1) {  // f32: a window's sum by itself, added with one rounding
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int term = PT - 1; term >= 0; --term) mma_f16(part, pa[0][term], b0, b1);
#pragma unroll
                    for (int y = 0; y < 4; ++y) o[0][j0 + j][y] += part[y];
                } else {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) mma_f16(o[mt][j0 + j], pa[mt][0], b0, b1);
                }
            }
            if (j0 + AHEAD * TJ < NJ) load_v(j0 + AHEAD * TJ);
        }
    };

    // Several warps per head meet at the end of a piece, at a barrier whose waits are bounded, too.  false: a wait gave up.
    uint32_t met = 0;
    auto meet = [&] {
        __syncwarp();
        if (lane == 0) mbar_arrive(s0 + (uint32_t)C::OFF_SYNC);
        return __all_sync(0xffffffffu, mbar_wait(s0 + (uint32_t)C::OFF_SYNC, met++ & 1)) != 0;
    };

    bool ok = true;
    for (int st = 0, at = 0, phase = 0;; st = st + 1 == STAGES ? 0 : st + 1, at = at + 1 == 2 * STAGES ? 0 : at + 1, phase ^= st == 0) {
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar_full + st * 8, phase)) != 0)) break;
        const Q8Stage* d = desc + at;
        const int4 what = *reinterpret_cast<const int4*>(d);
        const int k0 = what.x, sp = what.y, how = what.z;
        if (how < 0) break;
        if (how & Q8_ITEM)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                r[mt][0] = r[mt][1] = neg_inf();
                l[mt][0] = l[mt][1] = f2u(0.f, 0.f);
#pragma unroll
                for (int j = 0; j < NJ; ++j) o[mt][j][0] = o[mt][j][1] = o[mt][j][2] = o[mt][j][3] = 0.f;
            }
        if ((how & Q8_TURN) && !(ok = take_q())) break;

        const int first = k0 + kw;  // key of the warp's first column
        if (first < sp && first + KPW > 0) {
            const uint32_t kb = s0 + (uint32_t)(st * 2 * C::TENSOR), sc = s0 + (uint32_t)C::OFF_SC + (uint32_t)(st * 2 * C::SCALES * 4);
            if (first < 0 || first + KPW > least) window(std::true_type(), sp, first, kb, sc);
            else window(std::false_type(), sp, first, kb, sc);
        }

        if (!(how & Q8_LAST)) {
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + st * 8);
            continue;
        }
        // ---- the piece's result ----
        const int2 item = *reinterpret_cast<const int2*>(&d->pair);
        const Q8Tile tile = tile_of<PACKED>(p, ROWS, item.x);
        const int tile0 = tile.t * ROWS, h0 = item.y * p.hc;  // its first row, the group's first head
        const bool whole = (how & Q8_WHOLE) != 0;
        const size_t slot = ((size_t)c * 2 + (how & Q8_BEGIN ? 1 : 0)) * p.hc;
        float f[MT][2];
        float2 ml[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float sum, other;
                u2f(l[mt][y], sum, other);
                sum += other;
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                f[mt][y] = sum;
                if (wph > 1 && t == 0) {
                    const int row = mt * 16 + y * 8 + n;
                    sML[(wid * ROWS + row) * 2] = r[mt][y];
                    sML[(wid * ROWS + row) * 2 + 1] = sum;
                }
            }
        if (wph > 1 && !(ok = meet())) break;  // and every warp is done with the stage
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float m = r[mt][y], sum = f[mt][y];
                if (wph > 1) {
                    const int row = mt * 16 + y * 8 + n;
                    m = neg_inf();
                    for (int g = 0; g < wph; ++g) m = fmaxf(m, sML[((g * p.hc + hh) * ROWS + row) * 2]);
                    sum = 0.f;
                    for (int g = 0; g < wph; ++g) {
                        const float2 x = *reinterpret_cast<const float2*>(sML + ((g * p.hc + hh) * ROWS + row) * 2);
                        // a warp that saw nothing adds nothing; one whose reference is infinite has a NaN sum
                        sum += x.x == neg_inf() ? x.y : x.y * fast_exp2(x.x - m);
                    }
                }
                // a sum that is 0: nothing seen (or only NaN scores' zero weights, which make it NaN)
                const float inv = sum == 0.f ? 0.f : whole ? 1.f / sum : 1.f;
                f[mt][y] = r[mt][y] == neg_inf() && sum == sum ? 0.f : (wph > 1 && r[mt][y] != neg_inf() ? fast_exp2(r[mt][y] - m) * inv : inv);
                ml[mt][y] = make_float2(m, sum);
            }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int y = 0; y < 4; ++y) o[mt][j][y] *= f[mt][y >> 1];
        if (wph > 1) {
            // the warps of a head add up their outputs where the stage's K and V lay, half of them to the other half, a tile at a
            // time; a row's 8-column pieces are shuffled so that rows lie in different banks
            float* sO = reinterpret_cast<float*>(smem + (size_t)st * 2 * C::TENSOR);  // [hc][wph / 2][16][E]
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                for (int half = wph >> 1; half > 0 && ok; half >>= 1) {
                    float* part = sO + ((size_t)(hh * (wph >> 1) + (grp & (half - 1))) * 16 + n) * E + 2 * t;
                    if (grp >= half && grp < 2 * half)
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int y = 0; y < 2; ++y)
                                *reinterpret_cast<float2*>(part + 8 * y * E + 8 * (j ^ n)) = make_float2(o[mt][j][2 * y], o[mt][j][2 * y + 1]);
                    ok = meet();
                    if (grp < half)
#pragma unroll
                        for (int j = 0; j < NJ; ++j)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const float2 x = *reinterpret_cast<const float2*>(part + 8 * y * E + 8 * (j ^ n));
                                o[mt][j][2 * y] += x.x;
                                o[mt][j][2 * y + 1] += x.y;
                            }
                    if (half > 1 || mt + 1 < MT) ok = ok && meet();  // before they are written again
                }
            if (!ok) break;
            fence_proxy_async_smem();  // the next window is written here by TMA
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + st * 8);
        if (grp > 0) continue;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int i16 = mt * 16 + y * 8 + n, row = tile0 + i16;
                if (row >= tile.rows) continue;
                const int tok = row / p.G;
                const size_t orow = whole ? out_row<PACKED>(p, tile.tok0, (h0 + hh) * p.G + row - tok * p.G, tok) : (slot + hh) * ROWS + i16;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const float2 x = make_float2(o[mt][j][2 * y], o[mt][j][2 * y + 1]);
                    const size_t e = orow * E + 8 * j + 2 * t;
                    if (whole) {
                        store_pair<T>(static_cast<T*>(p.out) + e, x);
                        if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + e) = x;
                    } else {
                        *reinterpret_cast<float2*>(p.part_o + e) = x;
                    }
                }
                if (t == 0) {
                    if (!whole) p.part_ml[orow] = ml[mt][y];
                    else if (p.lse_out) p.lse_out[orow] = log_sum(ml[mt][y].x, ml[mt][y].y);
                }
            }
    }
    if (!ok && lane == 0) {  // a wait gave up
        *stop = 1;
        atomicOr(p.header + 3, 2);
    }
}

// ---- merge ----------------------------------------------------------------------------------
// Rows of items that more than one CTA worked on: their partials' sums, brought to one reference, in CTA
// order; zeros for pairs without a seen key; NaN in every output where the call's error word is set.
constexpr int kQ8Ahead = 4, kQ8MaxCtas = 1023;

// 2^x of a part's weight: ex2.approx is 2 ulp off, which shows in 32 bits.
template <class T> __device__ __forceinline__ float weight(float x) { return sizeof(T) == 4 ? exp2f(x) : fast_exp2(x); }

template <class T, int E, bool PACKED> __global__ void __launch_bounds__(256, 4) merge_q8_kernel(const __grid_constant__ Q8Params p, int rows, int ctas) {
    constexpr int TPR = E / 4, RPB = 256 / TPR;  // threads per row, rows per block
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, h = blockIdx.x % p.Hkv, pair = blockIdx.x / p.Hkv;
    const Q8Tile tile = tile_of<PACKED>(p, rows, pair);
    const int t = tile.t, hg = h / p.hc, hh = h - hg * p.hc;
    const float nan = __int_as_float(0x7fc00000);
    const long long P0 = __ldcg(p.P + pair), nw = __ldcg(p.P + pair + 1) - P0, first = P0 * p.hs + hg * nw;
    const bool failed = __ldcg(p.header + 3) != 0;
    int c0 = 0, c1 = -1;  // CTAs of the item: the last that begin at or before its first and last windows
    __shared__ long long starts[kQ8MaxCtas + 1];
    {
        long long at[(kQ8MaxCtas + 256) / 256];
#pragma unroll
        for (int x = 0; x < (kQ8MaxCtas + 256) / 256; ++x) at[x] = x * 256 + tid <= ctas ? __ldcg(p.cstart + x * 256 + tid) : 0;
#pragma unroll
        for (int x = 0; x < (kQ8MaxCtas + 256) / 256; ++x)
            if (x * 256 + tid <= ctas) starts[x * 256 + tid] = at[x];
        __syncthreads();
        auto last = [&](long long window) {  // CTA that begins at or before it, by a whole warp
            const int lane = tid & 31, g = 32 * (__popc(__ballot_sync(0xffffffffu, 32 * lane < ctas && starts[32 * lane & 1023] <= window)) - 1);
            return g + __popc(__ballot_sync(0xffffffffu, g + lane < ctas && starts[g + lane & 1023] <= window)) - 1;
        };
        if (nw > 0 && !failed) {
            c0 = last(first), c1 = last(first + nw - 1);
            if (c0 == c1) return;
        }
    }
    const int e = tid % TPR * 4;
    for (int i = blockIdx.y * RPB + tid / TPR; i < rows && t * rows + i < tile.rows; i += gridDim.y * RPB) {
        const int row = t * rows + i, s = row / p.G;
        const size_t orow = out_row<PACKED>(p, tile.tok0, h * p.G + row - s * p.G, s);
        float m = neg_inf(), den = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
        for (int c = c0; c <= c1; c += kQ8Ahead) {
            float2 x[kQ8Ahead];
            float4 v[kQ8Ahead];
#pragma unroll
            for (int k = 0; k < kQ8Ahead; ++k) {
                const size_t at = (((size_t)(c + k) * 2 + (c + k == c0 ? 1 : 0)) * p.hc + hh) * rows + i;
                x[k] = make_float2(neg_inf(), 0.f);
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (c + k <= c1 && starts[c + k] < starts[c + k + 1]) {  // a CTA may have no windows
                    x[k] = __ldcg(p.part_ml + at);
                    v[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * E + e));
                }
            }
            float mx = m;
#pragma unroll
            for (int k = 0; k < kQ8Ahead; ++k) mx = fmaxf(mx, x[k].x);
            const float mu = mx == neg_inf() ? 0.f : mx, alpha = weight<T>(m - mu);
            m = mx;
            den *= alpha;
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] *= alpha;
#pragma unroll
            for (int k = 0; k < kQ8Ahead; ++k) {
                if (x[k].y == 0.f) continue;  // an empty part adds nothing
                // a NaN sum: a NaN score (of a reference that is infinite, or of a row's only keys) reaches every element
                const float f = x[k].y != x[k].y ? x[k].y : weight<T>(x[k].x - mu);
                den = fmaf(f, x[k].y, den);
                a[0] = fmaf(f, v[k].x, a[0]);
                a[1] = fmaf(f, v[k].y, a[1]);
                a[2] = fmaf(f, v[k].z, a[2]);
                a[3] = fmaf(f, v[k].w, a[3]);
            }
        }
        const float inv = failed ? nan : den == 0.f ? 0.f : 1.f / den;
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] *= inv;
        store_quad<T>(static_cast<T*>(p.out) + orow * E + e, a[0], a[1], a[2], a[3]);
        if (p.out_f32) *reinterpret_cast<float4*>(p.out_f32 + orow * E + e) = make_float4(a[0], a[1], a[2], a[3]);
        if (p.lse_out && e == 0) p.lse_out[orow] = failed ? nan : log_sum(m, den);
    }
}

// ---- host side --------------------------------------------------------------------------------
namespace {

struct Q8Kernel {
    const void* fn[2];  // pages that come by TMA, row by row
    const void* rotate;
    const void* merge;
    int qhead, lims;        // bytes of a head's fragments and factors, of a tile's limits
    int krows, rows, ctas, heads, threads;  // CTAs per SM, KV heads of one at most
    size_t smem[2];
};
template <class T, int E, int MT, bool PACKED> Q8Kernel q8_kernel() {
    using C = Q8Cfg<T, E, MT, false>;
    using G = Q8Cfg<T, E, MT, true>;
    static_assert(C::KROWS == G::KROWS && C::CTAS == G::CTAS && C::HEADS == G::HEADS, "one layout");
    return {{(const void*)&decode_q8_kernel<T, E, MT, false, PACKED>, (const void*)&decode_q8_kernel<T, E, MT, true, PACKED>},
            (const void*)&rotate_q8_kernel<T, E, MT, PACKED>, (const void*)&merge_q8_kernel<T, E, PACKED>,
            C::QHEAD, C::LIMS, C::KROWS, C::ROWS, C::CTAS, C::HEADS, C::THREADS, {C::SMEM, G::SMEM}};
}
// One 16-row tile, or two where a KV head has more query rows (then the cache is read half as often); two
// tiles do not fit in the registers with 32-bit queries or head dim 256.
template <class T, bool PACKED> Q8Kernel q8_pick_t(int E, int rows) {
    if constexpr (sizeof(T) == 2)
        if (rows > 16 && E <= 128) return E == 64 ? q8_kernel<T, 64, 2, PACKED>() : q8_kernel<T, 128, 2, PACKED>();
    return E == 64 ? q8_kernel<T, 64, 1, PACKED>() : E == 128 ? q8_kernel<T, 128, 1, PACKED>() : q8_kernel<T, 256, 1, PACKED>();
}
template <bool PACKED> Q8Kernel q8_pick(int dtype, int E, int rows) {
    return dtype == DVATTN_FLOAT32   ? q8_pick_t<float, PACKED>(E, rows)
           : dtype == DVATTN_FLOAT16 ? q8_pick_t<__half, PACKED>(E, rows) : q8_pick_t<__nv_bfloat16, PACKED>(E, rows);
}

struct Q8Layout {
    size_t P, cstart, qf, ql, po, pl, total;
    int ctas, hc, nt, slice;  // slice: (sequence, row tile) pairs of a launch
    int items;                // of all
};
// Packed tokens: nseq sequences that begin at cu; `a` is the call with a token for a sequence.
struct Q8Packed {
    const int* cu;
    int nseq;
};
// By the query rows of a KV head in a sequence, of packed tokens on average (rounded up to whole tokens).  bf16, 64 / 8 heads of 128,
// two tiles against one: 592 packed sequences of one token behind 2000 keys 983 us against 578, 64 of them 135 against 82, 500 and a chunk
// of 256 tokens 944 against 602, 30 behind 8000 and a chunk of 28 222 against 149; head dim 64: 587 against 451, with a chunk 567
// against 474.  By the call's tokens, as without packing, all of these would have two.
Q8Kernel q8_of(const dvattn_paged_args* a, const Q8Packed* pk) {
    const int nseq = pk && pk->nseq > 0 ? pk->nseq : 1;
    const long long n = (pk ? ((long long)a->W + nseq - 1) / nseq : (long long)a->S) * (a->Hq / a->Hkv);
    const int rows = (int)(n < 1 << 20 ? n : 1 << 20);
    return pk ? q8_pick<true>(a->dtype, a->E, rows) : q8_pick<false>(a->dtype, a->E, rows);
}
int q8_layout(const dvattn_paged_args* a, const Q8Packed* pk, const Q8Kernel& k, Q8Layout& L) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return DVATTN_ERR_CUDA;
    L.ctas = sms * k.ctas < kQ8MaxCtas ? sms * k.ctas : kQ8MaxCtas;
    L.hc = a->Hkv % 4 == 0 && k.heads == 4 ? 4 : a->Hkv % 2 == 0 ? 2 : 1;
    L.nt = pk ? 1 : (a->S * (a->Hq / a->Hkv) + k.rows - 1) / k.rows;
    L.items = pk ? (int)((long long)a->W * (a->Hq / a->Hkv) / k.rows) + pk->nseq + 1 : a->W * L.nt;
    // 256 MB of fragments (one pair's, where that is more) keep the GPU busy: writing and reading them takes five times a launch's ends
    const long long fit = kQ8Fragments / ((long long)(a->F > 0 ? a->F : 1) * (a->Hkv * (long long)k.qhead + k.lims));
    L.slice = fit < 1 ? 1 : fit < kQ8MaxPairs ? (int)fit : kQ8MaxPairs;
    if (L.slice > L.nt) L.slice -= L.slice % L.nt;
    if (L.slice > L.items) L.slice = L.items;
    size_t at = 256;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    L.P = take(8 * ((size_t)L.slice + 1));
    L.cstart = take(8 * ((size_t)L.ctas + 1));
    L.qf = take((size_t)a->F * L.slice * a->Hkv * k.qhead);
    L.ql = take((size_t)a->F * L.slice * k.lims);
    L.po = take(4 * (size_t)L.ctas * 2 * L.hc * k.rows * a->E);
    L.pl = take(8 * (size_t)L.ctas * 2 * L.hc * k.rows);
    L.total = at;
    return DVATTN_OK;
}

int q8_validate(const dvattn_paged_args* a) {
    const int st = decode_validate(a);
    if (st != DVATTN_OK) return st;
    const long long rows = (long long)a->S * (a->Hq / a->Hkv);  // packed: of a token
    if (a->num_blocks < 0) return DVATTN_ERR_INVALID_ARGUMENT;
    // rows of a sequence; (turn, token)s, as many as row tiles or more; blocks of a launch
    if (rows > 32768 || (long long)(a->F > 0 ? a->F : 1) * a->W * a->S > 0x7fffffffLL || (long long)kQ8MaxPairs * a->Hkv * (a->F > 0 ? a->F : 1) > 0x7fffffffLL)
        return DVATTN_ERR_UNSUPPORTED;
    return DVATTN_OK;
}

// [tokens][Hkv][E] bytes as a 4-D map {128 (64) bytes, tokens, panels, heads} whose box is `box` tokens of hc heads,
// landing as [head][panel][token][128 (64) bytes], swizzled.
bool q8_map(CUtensorMap* m, const void* base, int E, int Hkv, int hc, long long tokens, int box) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint32_t rb = E < 128 ? 64 : 128;
    cuuint64_t dims[4] = {rb, (cuuint64_t)tokens, (cuuint64_t)(E / rb), (cuuint64_t)Hkv};
    cuuint64_t strides[3] = {(cuuint64_t)Hkv * E, rb, (cuuint64_t)E};
    cuuint32_t b[4] = {rb, (cuuint32_t)box, (cuuint32_t)(E / rb), (cuuint32_t)hc};
    cuuint32_t es[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              rb == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// DVATTN_TEST_STALL_TILE=<i>: tests only (see the decode launcher); read once per process.
int q8_stall_hook() {
    static const int t = [] {
        const char* e = getenv("DVATTN_TEST_STALL_TILE");
        return e && *e ? atoi(e) : -1;
    }();
    return t;
}

}  // namespace

static size_t q8_size(const dvattn_paged_args* a, const Q8Packed* pk) {
    if (q8_validate(a) != DVATTN_OK || (long long)a->W * a->S == 0 || a->Hq == 0) return 0;
    Q8Layout L;
    return q8_layout(a, pk, q8_of(a, pk), L) == DVATTN_OK ? L.total : 0;
}

static int q8_launch(const dvattn_paged_args* a, const Q8Packed* pk, const dvattn_q8_scales* sc, void* workspace, size_t wbytes, cudaStream_t stream) {
    int st = q8_validate(a);
    if (st != DVATTN_OK) return st;
    if (!sc) return DVATTN_ERR_INVALID_ARGUMENT;
    if ((long long)a->W * a->S == 0 || a->Hq == 0) return DVATTN_OK;
    const bool cached = a->max_blocks_per_seq > 0 && a->num_blocks > 0;
    if (!a->out || !a->queries || (a->F > 0 && (!a->locations || !a->fragment_lengths)) || (a->F > 0 && a->R > 0 && (!a->cosines || !a->sines)) ||
        (cached && (!a->k_cache || !a->v_cache || !a->block_tables || !sc->k_scales || !sc->v_scales)))
        return DVATTN_ERR_INVALID_ARGUMENT;
    for (const void* x : {a->queries, a->k_cache, a->v_cache, (const void*)a->out, (const void*)a->out_f32})
        if (reinterpret_cast<uintptr_t>(x) & 15) return DVATTN_ERR_INVALID_ARGUMENT;
    const Q8Kernel k = q8_of(a, pk);
    Q8Layout L;
    if ((st = q8_layout(a, pk, k, L)) != DVATTN_OK) return st;
    if (!workspace || wbytes < L.total || (reinterpret_cast<uintptr_t>(workspace) & 255)) return DVATTN_ERR_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    Q8Params p{};
    p.F = a->F; p.Hq = a->Hq; p.Hkv = a->Hkv; p.G = a->Hq / a->Hkv; p.S = a->S; p.R = a->R;
    p.rows = p.S * p.G;
    p.angles = pk ? a->R / 2 : a->R;
    p.cu = pk ? pk->cu : nullptr, p.nseq = pk ? pk->nseq : 0;
    p.BS = a->block_size; p.maxb = a->max_blocks_per_seq; p.NB = a->num_blocks;
    const long long cap = (long long)a->max_blocks_per_seq * a->block_size;
    p.cap = a->num_blocks <= 0 || (pk && pk->nseq == 0) ? 0 : cap > kMostPositions ? kMostPositions : (int)cap;
    p.hc = L.hc; p.hs = a->Hkv / L.hc; p.nt = L.nt;
    p.kt = k.krows / L.hc;
    p.tokens = (long long)a->W * a->S;
    p.scale_log2 = a->scale * kLog2e;
    p.out = a->out; p.lse_out = a->lse_out; p.out_f32 = a->out_f32;
    p.q = a->queries; p.cos = a->cosines; p.sin = a->sines; p.loc = a->locations; p.L = a->fragment_lengths;
    p.k = static_cast<const uint8_t*>(a->k_cache); p.v = static_cast<const uint8_t*>(a->v_cache);
    p.ks = sc->k_scales; p.vs = sc->v_scales; p.bt = a->block_tables;
    p.stall_tile = q8_stall_hook();
    p.header = reinterpret_cast<int*>(ws);
    uint8_t* qf = reinterpret_cast<uint8_t*>(ws + L.qf);
    uint8_t* ql = reinterpret_cast<uint8_t*>(ws + L.ql);
    p.qf = qf;
    p.ql = ql;
    p.P = reinterpret_cast<long long*>(ws + L.P);
    p.cstart = reinterpret_cast<long long*>(ws + L.cstart);
    p.part_o = reinterpret_cast<float*>(ws + L.po);
    p.part_ml = reinterpret_cast<float2*>(ws + L.pl);
    // pages that are whole numbers of boxes of 8 rows or more come by TMA, others row by row
    int box = p.kt;
    while (p.BS % box) box >>= 1;
    alignas(64) CUtensorMap mk{}, mv{};
    const bool gather = box < 8 || !cached || a->num_blocks * a->block_size > 0x7fffffffLL - 2 * box;
    if (gather) box = p.kt;
    else if (!q8_map(&mk, a->k_cache, a->E, a->Hkv, L.hc, a->num_blocks * a->block_size, box) ||
             !q8_map(&mv, a->v_cache, a->E, a->Hkv, L.hc, a->num_blocks * a->block_size, box))
        return DVATTN_ERR_CUDA;
    p.box = box;
    while (1 << p.box_shift < box) ++p.box_shift;
    p.align = gather ? 1 : box;
    p.bs_shift = (p.BS & (p.BS - 1)) == 0 ? 0 : -1;
    while (p.bs_shift >= 0 && 1 << p.bs_shift < p.BS) ++p.bs_shift;

    const void* fn = k.fn[gather];
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)k.smem[gather]) != cudaSuccess ||
        cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess)
        return DVATTN_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.stream = stream;
    cudaError_t e = cudaSuccess;
    for (long long x = 0; x < L.items && e == cudaSuccess; x += L.slice) {
        p.first = (int)x;
        p.pairs = L.items - p.first < L.slice ? L.items - p.first : L.slice;
        int rows = k.rows, ctas = L.ctas;
        void* rargs[] = {&p, &qf, &ql};
        cfg.gridDim = dim3((unsigned)((long long)a->F * p.pairs * a->Hkv));
        cfg.blockDim = dim3(128);
        cfg.dynamicSmemBytes = 0;
        if (a->F > 0) e = cudaLaunchKernelExC(&cfg, k.rotate, rargs);
        if (e != cudaSuccess) break;
        void* args[] = {&p, &mk, &mv};
        cfg.gridDim = dim3((unsigned)L.ctas);
        cfg.blockDim = dim3(k.threads);
        cfg.dynamicSmemBytes = k.smem[gather];
        cfg.numAttrs = a->F > 0 ? 1 : 0;  // it waits for nothing itself: the rotation has
        e = cudaLaunchKernelExC(&cfg, fn, args);
        cfg.numAttrs = 1;
        if (e != cudaSuccess) break;
        void* margs[] = {&p, &rows, &ctas};
        const int rpb = 256 / (a->E / 4);
        cfg.gridDim = dim3((unsigned)(p.pairs * a->Hkv), (unsigned)((rows + rpb - 1) / rpb));
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        e = cudaLaunchKernelExC(&cfg, k.merge, margs);
    }
    if (e != cudaSuccess) {
        if (getenv("DVATTN_DEBUG")) fprintf(stderr, "dvattn q8 launch: %s\n", cudaGetErrorString(e));
        return DVATTN_ERR_CUDA;
    }
    return cudaGetLastError() == cudaSuccess ? DVATTN_OK : DVATTN_ERR_CUDA;
}

size_t decode_q8_workspace_size(const dvattn_paged_args* a) { return q8_size(a, nullptr); }
int decode_q8_launch(const dvattn_paged_args* a, const dvattn_q8_scales* sc, void* workspace, size_t wbytes, cudaStream_t stream) {
    return q8_launch(a, nullptr, sc, workspace, wbytes, stream);
}
size_t packed_q8_workspace_size(const dvattn_paged_args* tokens, const int* cu, int nseq) {
    const Q8Packed pk{cu, nseq};
    return q8_size(tokens, &pk);
}
int packed_q8_launch(const dvattn_paged_args* tokens, const int* cu, int nseq, const dvattn_q8_scales* sc, void* workspace, size_t wbytes,
                     cudaStream_t stream) {
    const Q8Packed pk{cu, nseq};
    return q8_launch(tokens, &pk, sc, workspace, wbytes, stream);
}

}  // namespace dvb
