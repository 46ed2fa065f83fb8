// What the two sizes of the vocabulary cross entropy share: whole tiles of rows (vocab.hip) and few rows (vocab_few.hip).
#pragma once
#include "common.hpp"
#include "split.hpp"

namespace laya {

constexpr float LOG2E = 1.44269504088896341f;
// Rows that the few-row kernels take at most. Over 768 x 50368, both ways, theirs and on packed tiles: 129 rows 0.32 and
// 0.57 ms, 192 rows 0.35 and 0.59, 256 rows 0.53 and 0.60; 257 rows 0.69 on tiles. Their sums are held in registers, which
// hold no more.
constexpr int VOCAB_FEW = 256;

// Words of a call: labelled rows, targets outside the vocabulary, bits of max|w_t·x_t| and of max|W|, the ways that dx's
// sum and dW's are split, workgroups that have ended.
enum : int { WORD_COUNT, WORD_BAD, WORD_WX, WORD_W, WORD_SPLITS, WORD_SPLITS_E, WORD_ENDED, WORDS };

// Vector loads that ask for the elements' own alignment alone: the hardware takes them at any, so that a table of an odd
// width, or one that starts inside another array, reads as fast as an aligned one.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x8_any __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ void load8(const float* at, float (&v)[8]) {
    const f32x4_any a = *reinterpret_cast<const f32x4_any*>(at), b = *reinterpret_cast<const f32x4_any*>(at + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = a[i];
        v[4 + i] = b[i];
    }
}
__device__ __forceinline__ void load8(const __bf16* at, float (&v)[8]) {
    const bf16x8_any a = *reinterpret_cast<const bf16x8_any*>(at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
}
// Eight consecutive values of a row from column c, zeros behind K.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int c, int K, float (&v)[8]) {
    if (c + 8 <= K) {
        load8(row + c, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < K ? (float)row[c + i] : 0.0f;
    }
}

// The tiles' statistics part[tile][pitch] and the targets' logits into row_loss, lse and the weighted total.
void vocab_merge(laya_ctx* ctx, const VocabArgs& a, const float2* part, int pitch, int tiles, unsigned* words,
                 const int* row_of, const float* z_target, float* row_loss, float* lse, float* loss);
bool vocab_few_rows(const VocabArgs& a);
void vocab_few_fwd(laya_ctx* ctx, const VocabArgs& a, float* row_loss, float* lse, float* loss, int* bad_count);
void vocab_few_bwd(laya_ctx* ctx, const VocabArgs& a, const float* lse, float* dx, float* dW, float* db);

}  // namespace laya
