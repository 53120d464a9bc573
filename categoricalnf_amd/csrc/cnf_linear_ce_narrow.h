// Linear cross entropy of few features (H <= 128): the product over H fits the registers, so neither the logits nor their gradient
// leave the chip.  Interface between the kernels (cnf_linear_ce_narrow.hip) and the host side (cnf_linear_ce.hip).
#pragma once
#include "cnf_mfma.h"

namespace cnf {

constexpr float kLog2e = 1.4426950408889634f;

struct RowState {       // backward: what an element d = exp2(l log2 e - m2) scale - [target] g needs of its row
    float m2, scale;    // maximum times log2 e (+inf: the row is ignored); g / s
    float g;
    int target;         // -1: ignored
};

constexpr int kNarrowOwn = 128;         // rows (or vocabulary entries) of a workgroup
constexpr int kNarrowWalk = 64;         // vocabulary entries (or rows) of a step

struct NarrowArgs {
    Operand own, walk;                  // own: the side whose block a workgroup keeps in registers; walk: the side it goes through
    int hidden, vocab;
    int64_t rows;
    int splits;                         // of the walk
    const float* bias;                  // [vocabulary rounded up to kNarrowWalk] fp32, -inf behind the last entry
    // forward
    const int64_t* target;
    int64_t ignore;
    float2* partial;                    // [splits][rows]
    float* target_logit;                // [rows]
    // backward
    const RowState* state;              // [rows rounded up to kNarrowWalk]
    void* out;                          // final_dtype >= 0: [n][hidden] of that type; otherwise fp32 [splits][n][ld]
    int64_t ld;
    int final_dtype;
    const float* unscale;
    void* db;                           // nullable; partial sums: in column ld - 4 of out
    int db_dtype;
};

enum NarrowJob { kNarrowLse, kNarrowDx, kNarrowDw };

bool narrow_supported(int dtype, int hidden);
int narrow_launch(NarrowJob job, int dtype, const NarrowArgs& a, hipStream_t st);

}  // namespace cnf
