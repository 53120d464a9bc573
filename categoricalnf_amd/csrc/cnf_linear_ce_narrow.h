// Linear cross entropy of few features (H <= 128): the product over H fits the registers, so neither the logits nor their gradient
// leave the chip.  Interface between the kernels (cnf_linear_ce_narrow.hip) and the host side (cnf_linear_ce.hip).
#pragma once
#include "cnf_mfma.h"

namespace cnf {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

struct RowState {       // backward: what an element d = (exp2(l2 - m2) inv_s - [target]) g, l2 = l log2 e, needs of its row
    float m2, inv_s;    // maximum times log2 e (+inf: the row is ignored); 1 / s
    float g;            // over the largest |g|
    int target;         // -1: ignored
};

// Two fp16 parts of an operand scaled by one power of two hold 22 bits of what is above 2^-16 of its largest element, and 2^-39 of that
// largest of the rest.  An operand with a row whose largest element is below 2^-kRowSpan of the tensor's is "wide": its call takes the fp32
// matrix instructions (product32), so that no row's results depend on the size of the others.  14: a row at the border still has its
// 22 bits, and two are left for the sums over a vocabulary in which it alone has any probability.
constexpr int kRowSpan = 14;
// The gradient of the logits in fp16 (one part or two) is kept to 2^-39 of the largest |g|.  Where a row's |g| is that many powers of two
// below the largest, more than `apart`, its dx would be short of bits: dx applies g behind its product then; further than `plain` below
// (or beside an infinite or NaN g), fp32 operands take fp32 products, so that also a class that only such rows have gets its dw.  fp32:
// 2^-39 of the largest is 2^-27 of a row at `apart`, 2^-15 at `plain`; fp16: 2^-21 at 18, a few bits below d's own rounding.  The second pass
// over the logits takes 260 us of 1034 at 8192 x 8000 x 512 in fp32.
struct GradSpan {
    int apart, plain;
};
constexpr GradSpan kGradSpan32 = {12, 24}, kGradSpan16 = {18, 18};
constexpr int kWideMark = 4096;         // in an exponent that the forward hands to the backward: the operand is wide

// what the operands of a call were scaled by; in device memory
struct CeScales {
    int ex[2];          // fp32: x was multiplied by 2^ex[0], w by 2^ex[1]
    int wide[2];        // fp32: whether x, w are wide
    float top;          // largest |g|, or 1
    int wide_g;         // the rows' g: 0, 1: apart, 2: plain
};

constexpr int kNarrowOwn = 128;         // rows (or vocabulary entries) of a workgroup
constexpr int kNarrowWalk = 64;         // vocabulary entries (or rows) of a step

struct NarrowArgs {
    Operand own, walk;                  // own: the side whose block a workgroup keeps in registers; walk: the side it goes through
    int hidden, vocab;
    int64_t rows;
    int splits;                         // of the walk
    const float* bias;                  // [vocabulary rounded up to kNarrowWalk] fp32, times log2 e, -inf behind the last entry
    // forward
    const int64_t* target;
    int64_t ignore;
    float2* partial;                    // [splits][rows]; with one split the kernel finishes its rows itself:
    float* target_logit;                // [rows]
    float *row_max, *row_sum, *loss;    // [rows]
    double* sums;                       // [workgroups][2] sum and number of the rows that count
    float* reduced;                     // nullable: nobody asks for the sums; written by a single workgroup
    int* flags;
    // backward
    const RowState* state;              // [rows rounded up to kNarrowWalk]
    void* out;                          // final_dtype >= 0: [n][hidden] of that type; otherwise fp32 [splits][n][ld]
    int64_t ld;
    int final_dtype;
    const CeScales* scales;
    int scaled;                         // fp32 operands: scales->ex and ->wide hold
    Operand32 own32, walk32;            // the operands as they were given, for wide ones
    float lift;                         // d is computed times lift (a power of two): small probabilities stay normal numbers in fp16
    void* db;                           // nullable; partial sums: in column ld - 4 of out
    int db_dtype;
};

enum NarrowJob { kNarrowLse, kNarrowDx, kNarrowDw };

bool narrow_supported(int hidden);
int narrow_launch(NarrowJob job, int dtype, const NarrowArgs& a, hipStream_t st);

}  // namespace cnf
