// Float logits of few bf16 rows (few_bf16.hip).
#pragma once

#include "common.h"

// out [rows][tokens] (row stride ldo, a multiple of 4) = hidden weight^T for at most 64 rows;
// width a multiple of 64, rows of hidden and weight 16-byte aligned.
void few_bf16_logits(const bf16_t* hidden, int64_t ldh, const bf16_t* weight, int64_t ldw, int64_t rows,
                     int64_t tokens, int64_t width, float* out, int64_t ldo, hipStream_t st);
