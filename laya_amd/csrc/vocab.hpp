// What the two sizes of the vocabulary cross entropy share: whole tiles of rows (vocab.hip) and few rows (vocab_few.hip).
#pragma once
#include "common.hpp"
#include "split.hpp"

namespace laya {

constexpr float LOG2E = 1.44269504088896341f;
constexpr int VOCAB_FEW = 256;  // rows that the few-row kernels take at most

// Words of a call: labelled rows, targets outside the vocabulary, bits of max|w_t·x_t| and of max|W|, the ways that dx's
// sum is split, workgroups that have ended.
enum : int { WORD_COUNT, WORD_BAD, WORD_WX, WORD_W, WORD_SPLITS, WORD_ENDED, WORDS };

// Eight consecutive values of a row from column c, zeros behind K. VEC: rows start on 16 bytes and K is a multiple of 8.
template <bool VEC>
__device__ __forceinline__ void load8(const float* row, int c, int K, float (&v)[8]) {
    if constexpr (VEC) {
        const f32x4 zero = {};
        const f32x4 a = c < K ? *reinterpret_cast<const f32x4*>(row + c) : zero;
        const f32x4 b = c < K ? *reinterpret_cast<const f32x4*>(row + c + 4) : zero;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < K ? row[c + i] : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ void load8(const __bf16* row, int c, int K, float (&v)[8]) {
    if constexpr (VEC) {
        const bf16x8 zero = {};
        const bf16x8 a = c < K ? *reinterpret_cast<const bf16x8*>(row + c) : zero;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < K ? (float)row[c + i] : 0.0f;
    }
}

// The tiles' statistics part[tile][pitch] into row_loss, lse and the weighted total.
void vocab_merge(laya_ctx* ctx, const VocabArgs& a, const float2* part, int pitch, int tiles, unsigned* words,
                 const int* row_of, float* row_loss, float* lse, float* loss);
bool vocab_few_rows(const VocabArgs& a);
void vocab_few_fwd(laya_ctx* ctx, const VocabArgs& a, float* row_loss, float* lse, float* loss, int* bad_count);
void vocab_few_bwd(laya_ctx* ctx, const VocabArgs& a, const float* lse, float* dx, float* dW, float* db);

}  // namespace laya
