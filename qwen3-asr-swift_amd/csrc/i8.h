// Matrix products in 8-bit integers with a scale per activation row and per weight row (gfx950).
#pragma once
#include "common.h"

constexpr int I8_MAX_K = 131056;   // 127 * 127 * K stays below 2^31 with room to spare, also for -128 (128 * 128 * K)

struct I8Source {          // activations before they are rounded to 8 bits
    const void* x = nullptr;
    int f32 = 0;           // 0: bf16, 1: fp32
    int64_t ldx = 0;
};

struct I8Params {
    const int8_t* A = nullptr; int64_t lda = 0; const float* sa = nullptr;   // [M][lda], zero from K to the next multiple of 16
    const int8_t* W = nullptr; int64_t ldw = 0; const float* sw = nullptr;   // [N][ldw]
    const float* bias = nullptr;
    int M = 0, N = 0, K = 0;
    void* out = nullptr; int64_t ldo = 0; int out_f32 = 0;
};

void launch_i8_quantize(const I8Source& src, int rows, int cols, int8_t* q, int64_t ldq, float* scales, hipStream_t s);
// Both steps in one kernel where the rows are few; false: it does not apply.
bool launch_i8_linear_few_rows(const I8Params& p, const I8Source& src, hipStream_t s);
void launch_i8_matmul(const I8Params& p, hipStream_t s);
