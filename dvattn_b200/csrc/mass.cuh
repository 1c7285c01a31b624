// What the attention-mass kernels share (mass.cu, mass_tc.cu).
#pragma once

#include <cuda.h>

#include "turns.cuh"

namespace dvb {

struct MassParams : TurnSplit {
    int Hq, Hkv, G, S, R;
    int rows, rows_pad;  // S * G queries of a KV head: row r = (query r / G, head r % G); a multiple of 16
    int passes;          // row tiles that a CTA runs one after the other over its windows (mass_tc.cu)
    int rot_vec;         // rotary halves are whole 16-byte chunks, cos/sin rows 16-byte aligned
    int box;             // rows of a TMA box, 0: rows are gathered
    int stall_tile;      // test hook (DVATTN_TEST_STALL_TILE), -1: off
    long long N;         // positions of a mass row
    float scale_log2;
    float* mass;
    const float* lse;
    const void* q;
    const float* cos;
    const float* sin;
    const void* k;
    // workspace; a row past `rows`, or whose lse is -inf, gives no weight: its query is that of a row
    // that does (zeros where none does), its nlse the lowest number, its lim 0
    int* header;  // [3] error word (kErrorWordOffset)
    void* qr;     // [F][W][Hkv][rows_pad][E] T, queries rotated for the turn
    float* nlse;  // [W][Hkv][rows_pad] -lse in log2 units
    int* lim;     // [F][W][Hkv][rows_pad] keys of the turn that the row sees
    int* all;     // [F][W][Hkv] keys of the turn that every row sees that gives weight
};

struct MassMaps {
    CUtensorMap q, k;
};
struct MassKernel {
    const void* fn;
    int threads, kt, ctas;
    int pass_rows;  // rows of a pass
    size_t smem;
};
// the 16-bit kernel on the 5th-generation tensor cores (mass_tc.cu), and its tensor maps
MassKernel mass_tc_pick(int dtype, int E, int rows);
bool mass_tc_maps(MassParams& p, int dtype, int E, MassMaps& maps);

}  // namespace dvb
