// Float32 products of few rows with a weight [vocab, width] that is read or written once
// (few_f32.hip).
#pragma once

#include "common.h"

constexpr int64_t FEW_F32_ROWS = 32;
// Rows of D as the kernels read it: D [tokens][few_f32_pad(rows)], tokens first.
int64_t few_f32_pad(int64_t rows);
// Parts of the tokens that few_f32_hidden leaves planes of.
int64_t few_f32_planes(int64_t tokens, int64_t width);
// planes [few_f32_planes][rows][width] whose sum is D^T weight.
void few_f32_hidden(const float* D, const float* weight, int64_t ldw, int64_t rows, int64_t tokens,
                    int64_t width, float* planes, hipStream_t st);
// out [tokens][width] = D hidden, rows of hidden 16-byte aligned.
void few_f32_weight(const float* D, const float* hidden, int64_t ldh, int64_t rows, int64_t tokens,
                    int64_t width, float* out, hipStream_t st);
