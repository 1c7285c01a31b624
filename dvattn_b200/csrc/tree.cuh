// What the draft-tree attention kernels share: the call's parameters.
//
// A call attends, for every sequence w, the S tokens of a drafted tree over the sequence's
// cached turns and over the tree itself: token s sees the cached keys its locations let it
// see and the drafted keys of its ancestors (and its own).  All S * G query rows of a KV
// head (row r = token r / G, head r % G of the group) read the same keys, so an item is
// (w, row tile of `mi` rows, KV head), and its windows (turns.cuh) end with the drafted
// keys.  A CTA's range that starts or ends inside an item leaves a partial result (two slots
// per CTA: 0 for the piece that continues an item, 1 for the piece that starts one), merged
// by tree_merge_kernel.
#pragma once

#include <cuda.h>

#include "turns.cuh"

namespace dvb {

struct TreeParams : TurnSplit {
    int Hq, Hkv, G, S, R;
    int SW;  // 32-bit words of a token's ancestor set, a multiple of 4
    int mi;  // rows per item
    int box;  // rows of a TMA box (pages and windows are whole numbers of boxes); 0: rows are gathered
    int rot_vec;     // rotary halves are whole 16-byte chunks, cos/sin rows 16-byte aligned
    int rows;        // S * G query rows of a KV head
    int out_sectors; // the output is 32-byte aligned
    int stall_tile;  // test hook (DVATTN_TEST_STALL_TILE), -1: off
    float scale_log2;
    void* out;
    float* lse_out;
    const void* q;
    const float* cos;
    const float* sin;
    const int* parents;
    const void* k;
    const void* v;
    const void* dk;
    const void* dv;
    // workspace
    int* header;      // [2] a value of the call is odd (below); [3] error word (kErrorWordOffset)
    uint32_t* anc;    // [W][S][SW] ancestor sets; a token that is not there has an empty one
    int* lim;         // [F][W][S] keys of the turn that the token sees; 0: it is not there
    int* same;        // [W][F] keys of the turn that every token sees that is there
    // values that are not finite (16-bit types: tree_merge_kernel)
    uint8_t* odd;     // [W][Hkv][S] the drafted value is odd: it has an infinity or NaN
    int* odd_any;     // [W][Hkv] so has one of them, or a cached value in the windows that are looked through
    void* dvr;        // [W][Hkv][S][E] T, drafted values with zeros for such elements
    void* dkr;        // [W][Hkv][S][E] T, drafted keys rotated
    void* qr;         // [F][W][Hkv][rows][E] T, queries rotated for the turn
    float* part_o;    // [CTAs][2][mi][E] normalised partial outputs
    float* part_lse;  // [CTAs][2][mi] log2 sums, -inf: nothing seen
};

// An attention kernel and its launch shape.
struct TreeKernel {
    const void* fn;
    int threads, kt, mi;
    int ctas;   // per SM
    int least;  // windows a CTA group has at least
    size_t smem;
};
// the 16-bit kernel on the 5th-generation tensor cores (tree_tc.cu), and its tensor maps
struct TreeMaps {
    CUtensorMap q, k, v, dk, dv;
};
TreeKernel tree_tc_pick(int dtype, int E, int rows);
// Sets p.box and p.align and fills the maps the kernel then uses; false: a CUDA error.
bool tree_tc_maps(TreeParams& p, int dtype, int E, TreeMaps& maps);

}  // namespace dvb
