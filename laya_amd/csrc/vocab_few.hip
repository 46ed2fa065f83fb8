// The vocabulary cross entropy of up to 128 rows, where the table's own bytes are the cost: every kernel reads W (or
// moves dW) once, straight from memory, and splits it in registers.
//
// The products are exact three-piece bf16 splits (split.hpp): six matrix products for one, but no scale, and so no pass
// over W to find one; up to 128 rows their time hides behind the table's. bf16 weights are one piece, three products.
//   few_prepare   the labelled rows' x as fragments, rows t over h and (weighted) rows h over t
//   few_logits    z = W·xᵀ, a wave 16 rows of W (its 8 k of a lane are two 16-byte loads); statistics, or G in both orders
//   few_dx        dxᵀ = Wᵀ·Gᵀ over slices of the vocabulary, a lane's 8 k eight loads down W's column
//   few_dw        dWᵀ += xᵀ·G, a lane four neighbours of one row of dW
// Fragments are 16 rows x 32 k of v_mfma_f32_16x16x32_bf16, [k / 8][row][8 k], three planes one after another.
#include "elementwise.hpp"
#include "packed.hpp"
#include "vocab.hpp"

namespace laya {
namespace {

using packed::FRAG;
using packed::lds_byte;

constexpr int FEW_V = 128;  // rows of W a workgroup of few_logits takes

__device__ __forceinline__ void split8(const float (&v)[8], bf16x8 (&p)[3]) {
    bf16x4 a[3], b[3];
    split3_4(f32x4{v[0], v[1], v[2], v[3]}, a[0], a[1], a[2]);
    split3_4(f32x4{v[4], v[5], v[6], v[7]}, b[0], b[1], b[2]);
#pragma unroll
    for (int k = 0; k < 3; ++k) p[k] = __builtin_shufflevector(a[k], b[k], 0, 1, 2, 3, 4, 5, 6, 7);
}
// c += a·b of three-piece operands (PA = 1: a is one piece), smallest products first.
template <int PA>
__device__ __forceinline__ void mma(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x4& c) {
    if constexpr (PA == 3) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[2], b[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[0], c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[2], c, 0, 0, 0);
    }
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ bf16x8 fragment(const __bf16* at, int lane) {
    return *reinterpret_cast<const bf16x8*>(at + lane * 8);
}

// The labelled rows in order, by every workgroup for itself: row_of[j] (LDS) and their number. Rows ≤ VOCAB_FEW ≤ 256.
__device__ __forceinline__ int list_rows(const int* targets, int rows, int vocab, int* row_of, int& bad) {
    __shared__ int wave_count[4], wave_bad[4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int y = tid < rows ? targets[tid] : LAYA_NO_LABEL;
    const bool has = tid < 256 && y >= 0 && y < vocab;
    const unsigned long long m = __ballot(has), wrong = __ballot(tid < 256 && !has && y != LAYA_NO_LABEL);
    if (lane == 0 && wave < 4) {
        wave_count[wave] = __popcll(m);
        wave_bad[wave] = __popcll(wrong);
    }
    __syncthreads();
    int before = 0, count = 0;
    bad = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += wave_count[w];
        count += wave_count[w];
        bad += wave_bad[w];
    }
    if (has) row_of[before + __popcll(m & ((1ull << lane) - 1))] = tid;
    __syncthreads();
    return count;
}

struct Prepare {
    const float *x, *weights;
    const int* targets;
    int rows, hidden, vocab, blocks_t;  // blocks_t: blocks of 16 rows, padded
    __bf16* x_rows;                     // [k step][block of t][3][FRAG]
    __bf16* x_cols;                     // [block of 16 h][step of 32 t][3][FRAG], weighted (null: not wanted)
    int *row_of, *place, *bad_count;
    unsigned* words;
    float *row_loss, *lse;              // of the forward (null in the backward)
};

// One workgroup a step of 32 columns of x.
__global__ __launch_bounds__(256) void few_prepare_kernel(Prepare p) {
    __shared__ int row_of[256];
    __shared__ float tile[32][33];
    const int tid = threadIdx.x, step = blockIdx.x;
    int bad;
    const int count = list_rows(p.targets, p.rows, p.vocab, row_of, bad);
    if (step == 0) {
        if (tid < WORDS) p.words[tid] = tid == WORD_COUNT ? count : tid == WORD_BAD ? bad : 0;
        if (tid == 0 && p.bad_count) *p.bad_count = bad;
        if (tid < p.rows) {
            const int y = p.targets[tid];
            const bool has = y >= 0 && y < p.vocab;
            if (!has && p.row_loss) p.row_loss[tid] = p.lse[tid] = 0.0f;
            if (!has && p.place) p.place[tid] = -1;
        }
        if (tid < count) {
            p.row_of[tid] = row_of[tid];
            if (p.place) p.place[row_of[tid]] = tid;
        }
    }
    const int steps_t = (p.blocks_t + 1) / 2;
    for (int s = 0; s < steps_t; ++s) {  // 32 rows of x at a time: thread t four columns of row t / 8
        const int j = 32 * s + (tid >> 3), c = 32 * step + 4 * (tid & 7);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            tile[tid >> 3][4 * (tid & 7) + i] =
                j < count && c + i < p.hidden ? p.x[(size_t)row_of[j] * p.hidden + c + i] : 0.0f;
        __syncthreads();
        if (tid >= 128) continue;  // unit tid: row r, octet o
        float v[8];
        bf16x8 f[3];
        const int r = tid >> 2, o = tid & 3;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[r][8 * o + i];
        split8(v, f);
        const int tb = 2 * s + (r >> 4);
        if (tb < p.blocks_t) {
            __bf16* to = p.x_rows + ((size_t)step * p.blocks_t + tb) * (3 * FRAG) + (o * 16 + (r & 15)) * 8;
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(to + k * FRAG) = f[k];
        }
        if (p.x_cols) {  // row r of this side: column 32·step + r of x, over t
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = 32 * s + 8 * o + i;
                v[i] = t < count ? tile[8 * o + i][r] * (p.weights ? p.weights[row_of[t]] : 1.0f) : 0.0f;
            }
            split8(v, f);
            __bf16* to = p.x_cols + ((size_t)(2 * step + (r >> 4)) * steps_t + s) * (3 * FRAG) + (o * 16 + (r & 15)) * 8;
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(to + k * FRAG) = f[k];
        }
    }
}

// ------------------------------------------------------------------------------------------- shared

// Fragments that all waves of a workgroup read, copied to an LDS ring a step at a time: NB·3 KB in a row a step, each
// wave starting PER copies of 1 KB (the last ones may repeat one: the same bytes to the same place).
template <int NB, int WAVES, int RING>
struct Stream {
    static constexpr int KB = 3 * NB, PER = (KB + WAVES - 1) / WAVES, STEP = KB * FRAG;
    const __bf16* from;
    unsigned lds0;
    int chunk[PER], last;
    __device__ __forceinline__ Stream(const __bf16* data, const __bf16* lds, int wave, int lane, int steps)
        : from(data + lane * 8), lds0(lds_byte(lds)), last(steps - 1) {
#pragma unroll
        for (int k = 0; k < PER; ++k) chunk[k] = __builtin_amdgcn_readfirstlane(min(wave + k * WAVES, KB - 1));
    }
    // Step s into its slot; past the end the last step again, so that each step has as many copies under way.
    __device__ __forceinline__ void start(int s) const {
        const size_t at = (size_t)min(s, last) * STEP;
        const unsigned slot = lds0 + (unsigned)(s % RING) * (2 * STEP);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const unsigned to = slot + chunk[k] * (2 * FRAG);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to),
                         "v"(from + at + chunk[k] * FRAG) : "memory");
        }
    }
};

// ------------------------------------------------------------------------------------------- logits

struct FewLogits {
    const void* W;
    const float* bias;
    const __bf16* x_rows;
    const unsigned* words;
    int hidden, vocab, steps;
    // Statistics:
    float2* part;            // [tile of FEW_V][pitch]
    int pitch;
    // G:
    const int *row_of, *targets;
    const float *lse, *weights;
    __bf16* g_rows;          // [step of 32 v][block of t][3][FRAG]: rows t over v
    __bf16* g_cols;          // [block of 16 v][step of 32 t][3][FRAG]: rows v over t
    float* db;
    float scale;
};

constexpr int AHEAD = 4;  // steps of W that a wave has under way

template <int NB, typename TW, bool VEC, bool GRAD>
__global__ __launch_bounds__(512, 2) void few_logits_kernel(FewLogits p) {
    constexpr int PW = sizeof(TW) == 2 ? 1 : 3, RING = 4;
    typedef Stream<NB, 8, RING> S;
    __shared__ __attribute__((aligned(16))) __bf16 lds[RING * S::STEP < 16384 ? 16384 : RING * S::STEP];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, steps = p.steps;
    const int v0 = blockIdx.x * FEW_V + wave * 16;
    const TW* row = static_cast<const TW*>(p.W) + (size_t)min(v0 + (lane & 15), p.vocab - 1) * p.hidden;
    const S x(p.x_rows, lds, wave, lane, steps);
    float w[AHEAD][8];
    f32x4 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = f32x4{};
#pragma unroll
    for (int k = 0; k < RING - 1; ++k) x.start(k);
#pragma unroll
    for (int k = 0; k < AHEAD - 1; ++k) load8<VEC>(row, 32 * k + 8 * (lane >> 4), p.hidden, w[k]);
    auto step = [&](int s, auto slot) {
        constexpr int K = decltype(slot)::value;
        // Step s's copies have landed for every wave, and step s − 1 is read by all: its slot is free.
        packed::wait_copies<0>();
        x.start(s + RING - 1);
        load8<VEC>(row, 32 * (s + AHEAD - 1) + 8 * (lane >> 4), p.hidden, w[(K + AHEAD - 1) % AHEAD]);
        bf16x8 a[3];
        split8(w[K], a);
        const __bf16* xs = lds + K * S::STEP;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            bf16x8 b[3];
#pragma unroll
            for (int q = 0; q < 3; ++q) b[q] = fragment(xs + (3 * j + q) * FRAG, lane);
            mma<PW>(a, b, acc[j]);
        }
    };
    for (int s = 0; s < steps; s += 4) {
        step(s, std::integral_constant<int, 0>());
        if (s + 1 < steps) step(s + 1, std::integral_constant<int, 1>());
        if (s + 2 < steps) step(s + 2, std::integral_constant<int, 2>());
        if (s + 3 < steps) step(s + 3, std::integral_constant<int, 3>());
    }
    packed::wait_copies<0>();
    const int count = (int)p.words[WORD_COUNT];
    float b[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int v = v0 + 4 * (lane >> 4) + r;
        b[r] = v < p.vocab ? (p.bias ? p.bias[v] : 0.0f) : -__builtin_inff();
    }
    if constexpr (!GRAD) {
        float2* red = reinterpret_cast<float2*>(lds);  // [wave][16·NB]
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float m = -__builtin_inff(), s = 0.0f, z[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                z[r] = acc[j][r] + b[r];
                m = fmaxf(m, z[r]);
            }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float at = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
            for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((z[r] - at) * LOG2E);
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            if (lane < 16) red[wave * (16 * NB) + 16 * j + lane] = make_float2(m, s);
        }
        __syncthreads();
        if (tid < 16 * NB) {
            float m = -__builtin_inff(), s = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) m = fmaxf(m, red[q * (16 * NB) + tid].x);
            const float at = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float2 a = red[q * (16 * NB) + tid];
                s += a.y * __builtin_amdgcn_exp2f((a.x - at) * LOG2E);
            }
            p.part[(size_t)blockIdx.x * p.pitch + tid] = make_float2(m, s);
        }
    } else {
        constexpr int PITCH = 36, STEPS_T = (NB + 1) / 2;
        float* turn = reinterpret_cast<float*>(lds) + wave * (16 * PITCH);
        f32x4 db = {};
#pragma unroll
        for (int ts = 0; ts < STEPS_T; ++ts) {
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const int j = 2 * ts + jj, t = 16 * j + (lane & 15);
                f32x4 g = {};
                if (j < NB) {
                    const bool live = t < count;
                    const int r = live ? p.row_of[t] : 0;
                    const float lse = live ? p.lse[r] : 0.0f;
                    const int y = (live ? p.targets[r] : -1) - (v0 + 4 * (lane >> 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float q = __builtin_amdgcn_exp2f((acc[j][e] + b[e] - lse) * LOG2E);
                        q -= y == e ? 1.0f : 0.0f;
                        g[e] = live ? q : 0.0f;
                    }
                    const float wt = live ? (p.weights ? p.weights[r] : 1.0f) : 0.0f;
                    db += live ? g * wt : f32x4{};
                    bf16x4 f[3];
                    split3_4(g, f[0], f[1], f[2]);
                    __bf16* to = p.g_rows + ((size_t)(v0 >> 5) * NB + j) * (3 * FRAG) +
                                 (((wave & 1) * 2 + (lane >> 5)) * 16 + (lane & 15)) * 8 + 4 * ((lane >> 4) & 1);
#pragma unroll
                    for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x4*>(to + q * FRAG) = f[q];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) turn[(4 * (lane >> 4) + e) * PITCH + 16 * jj + (lane & 15)] = g[e];
            }
            float v[8];
            bf16x8 f[3];
            const float* at = turn + (lane & 15) * PITCH + 8 * (lane >> 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = at[e];
            split8(v, f);
            __bf16* to = p.g_cols + ((size_t)(v0 >> 4) * STEPS_T + ts) * (3 * FRAG) + lane * 8;
#pragma unroll
            for (int q = 0; q < 3; ++q) *reinterpret_cast<bf16x8*>(to + q * FRAG) = f[q];
        }
        if (p.db) {
#pragma unroll
            for (int o = 1; o < 16; o <<= 1)
#pragma unroll
                for (int e = 0; e < 4; ++e) db[e] += __shfl_xor(db[e], o, 64);
            const int v = v0 + 4 * (lane >> 4);
            if ((lane & 15) == 0)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (v + e < p.vocab) p.db[v + e] += db[e] * p.scale;
        }
    }
}

// -------------------------------------------------------------------------------------------- dx

struct FewDx {
    const void* W;
    const __bf16* g_rows;
    int hidden, vocab, steps, per;  // steps of 32 v in all, and of a slice
    float* part;                    // [slice][16·NB][hidden]
};

// A workgroup: 256 columns of W (a wave 32) over a slice of the vocabulary.
template <int NB, typename TW>
__global__ __launch_bounds__(512, 1) void few_dx_kernel(FewDx p) {
    constexpr int PW = sizeof(TW) == 2 ? 1 : 3, RING = 4;
    typedef Stream<NB, 8, RING> S;
    __shared__ __attribute__((aligned(16))) __bf16 lds[RING * S::STEP];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = blockIdx.y * p.per, steps = min(p.per, p.steps - first);
    const int h0 = blockIdx.x * 256 + wave * 32;
    const TW* W = static_cast<const TW*>(p.W);
    const S g(p.g_rows + (size_t)first * S::STEP, lds, wave, lane, steps);
    int col[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) col[i] = min(h0 + 16 * i + (lane & 15), p.hidden - 1);
    // Rows behind the vocabulary read its last: G is zero there.
    auto load = [&](int s, float (&w)[2][8]) {
        const int v = 32 * (first + min(s, steps - 1)) + 8 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[i][e] = (float)W[(size_t)min(v + e, p.vocab - 1) * p.hidden + col[i]];
    };
    float w[AHEAD][2][8];
    f32x4 acc[2][NB];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{};
#pragma unroll
    for (int k = 0; k < RING - 1; ++k) g.start(k);
#pragma unroll
    for (int k = 0; k < AHEAD - 1; ++k) load(k, w[k]);
    auto step = [&](int s, auto slot) {
        constexpr int K = decltype(slot)::value;
        packed::wait_copies<0>();
        g.start(s + RING - 1);
        load(s + AHEAD - 1, w[(K + AHEAD - 1) % AHEAD]);
        bf16x8 a[2][3];
        split8(w[K][0], a[0]);
        split8(w[K][1], a[1]);
        const __bf16* gs = lds + K * S::STEP;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            bf16x8 b[3];
#pragma unroll
            for (int q = 0; q < 3; ++q) b[q] = fragment(gs + (3 * j + q) * FRAG, lane);
            mma<PW>(a[0], b, acc[0][j]);
            mma<PW>(a[1], b, acc[1][j]);
        }
    };
    for (int s = 0; s < steps; s += 4) {
        step(s, std::integral_constant<int, 0>());
        if (s + 1 < steps) step(s + 1, std::integral_constant<int, 1>());
        if (s + 2 < steps) step(s + 2, std::integral_constant<int, 2>());
        if (s + 3 < steps) step(s + 3, std::integral_constant<int, 3>());
    }
    packed::wait_copies<0>();
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        float* to = p.part + ((size_t)blockIdx.y * (16 * NB) + 16 * j + (lane & 15)) * p.hidden;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int h = h0 + 16 * i + 4 * (lane >> 4) + e;
                if (h < p.hidden) to[h] = acc[i][j][e];
            }
    }
}

// dx_r = w_r·scale·Σ over the slices, 0 for rows without a label.
__global__ __launch_bounds__(256) void few_dx_sum_kernel(const float* __restrict__ part, int slices, int pitch,
                                                         const int* __restrict__ place,
                                                         const float* __restrict__ weights, float scale, int hidden,
                                                         float* __restrict__ dx) {
    const int r = blockIdx.y, h = blockIdx.x * 256 + threadIdx.x, j = place[r];
    if (h >= hidden) return;
    float s[4] = {};
    if (j >= 0) {
        const float* at = part + (size_t)j * hidden + h;
        const size_t next = (size_t)pitch * hidden;
        int k = 0;
        for (; k + 3 < slices; k += 4)
#pragma unroll
            for (int q = 0; q < 4; ++q) s[q] += at[(k + q) * next];
        for (; k < slices; ++k) s[0] += at[k * next];
    }
    dx[(size_t)r * hidden + h] = j >= 0 ? ((s[0] + s[1]) + (s[2] + s[3])) * (weights ? weights[r] : 1.0f) * scale : 0.0f;
}

// -------------------------------------------------------------------------------------------- dW

struct FewDw {
    const __bf16 *x_cols, *g_cols;
    const unsigned* words;
    int hidden, vocab;
    float scale;
    float* dW;
};

// A wave: 16 rows of dW, their G in registers, all blocks of 16 columns one after another.
template <int STEPS_T, bool VEC>
__global__ __launch_bounds__(256) void few_dw_kernel(FewDw p) {
    if (p.words[WORD_COUNT] == 0) return;
    constexpr int FETCH = 4;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, vb = blockIdx.x * 4 + wave;
    const int v = 16 * vb + (lane & 15), blocks = (p.hidden + 15) / 16;
    if (16 * vb >= p.vocab) return;
    bf16x8 g[STEPS_T][3];
#pragma unroll
    for (int s = 0; s < STEPS_T; ++s)
#pragma unroll
        for (int q = 0; q < 3; ++q) g[s][q] = fragment(p.g_cols + (((size_t)vb * STEPS_T + s) * 3 + q) * FRAG, lane);
    float* row = p.dW + (size_t)min(v, p.vocab - 1) * p.hidden;
    const bool live = v < p.vocab;
    auto fetch = [&](int hb) {
        const int h = 16 * min(hb, blocks - 1) + 4 * (lane >> 4);
        f32x4 o = {};
        if constexpr (VEC) {
            o = *reinterpret_cast<const f32x4*>(row + h);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = row[min(h + e, p.hidden - 1)];
        }
        return o;
    };
    f32x4 old[FETCH];
#pragma unroll
    for (int k = 0; k < FETCH; ++k) old[k] = fetch(k);
    for (int hb = 0; hb < blocks; hb += FETCH)
#pragma unroll
        for (int k = 0; k < FETCH; ++k) {
            if (hb + k >= blocks) break;
            const __bf16* xs = p.x_cols + (size_t)(hb + k) * STEPS_T * (3 * FRAG);
            f32x4 c = {};
#pragma unroll
            for (int s = 0; s < STEPS_T; ++s) {
                bf16x8 a[3];
#pragma unroll
                for (int q = 0; q < 3; ++q) a[q] = fragment(xs + (s * 3 + q) * FRAG, lane);
                mma<3>(a, g[s], c);
            }
            const f32x4 now = old[k] + c * p.scale;
            old[k] = fetch(hb + k + FETCH);
            const int h = 16 * (hb + k) + 4 * (lane >> 4);
            if (!live) continue;
            if constexpr (VEC) {
                *reinterpret_cast<f32x4*>(row + h) = now;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (h + e < p.hidden) row[h + e] = now[e];
            }
        }
}

// ------------------------------------------------------------------------------------------ launches

int blocks_of(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }

template <int NB, bool GRAD>
void launch_logits(laya_ctx* ctx, const VocabArgs& a, const FewLogits& p) {
    const dim3 grid((a.vocab + FEW_V - 1) / FEW_V), block(512);
    const bool vec = a.hidden % 8 == 0 && ((uintptr_t)p.W & 15u) == 0;
    ProfileScope scope(ctx, "vocab_few_logits", 2.0 * a.rows * a.hidden * a.vocab,
                       (a.W16 ? 2.0 : 4.0) * a.hidden * a.vocab);
    if (a.W16 && vec)
        LAYA_LAUNCH((few_logits_kernel<NB, __bf16, true, GRAD>), grid, block, 0, ctx->stream, p);
    else if (a.W16)
        LAYA_LAUNCH((few_logits_kernel<NB, __bf16, false, GRAD>), grid, block, 0, ctx->stream, p);
    else if (vec)
        LAYA_LAUNCH((few_logits_kernel<NB, float, true, GRAD>), grid, block, 0, ctx->stream, p);
    else
        LAYA_LAUNCH((few_logits_kernel<NB, float, false, GRAD>), grid, block, 0, ctx->stream, p);
    check_launch("few_logits_kernel");
}
template <bool GRAD>
void launch_logits(laya_ctx* ctx, const VocabArgs& a, const FewLogits& p, int nb) {
    if (nb == 1) launch_logits<1, GRAD>(ctx, a, p);
    else if (nb == 2) launch_logits<2, GRAD>(ctx, a, p);
    else if (nb == 4) launch_logits<4, GRAD>(ctx, a, p);
    else launch_logits<8, GRAD>(ctx, a, p);
}

template <int NB>
void launch_dx(laya_ctx* ctx, const VocabArgs& a, const FewDx& p, int slices) {
    const dim3 grid((a.hidden + 255) / 256, slices), block(512);
    if (a.W16)
        LAYA_LAUNCH((few_dx_kernel<NB, __bf16>), grid, block, 0, ctx->stream, p);
    else
        LAYA_LAUNCH((few_dx_kernel<NB, float>), grid, block, 0, ctx->stream, p);
    check_launch("few_dx_kernel");
}

template <int STEPS_T>
void launch_dw(laya_ctx* ctx, const VocabArgs& a, const FewDw& p) {
    const dim3 grid((a.vocab + 63) / 64), block(256);
    ProfileScope scope(ctx, "vocab_few_dw", 2.0 * a.rows * a.hidden * a.vocab, 8.0 * a.hidden * a.vocab);
    if (a.hidden % 16 == 0 && ((uintptr_t)p.dW & 15u) == 0)
        LAYA_LAUNCH((few_dw_kernel<STEPS_T, true>), grid, block, 0, ctx->stream, p);
    else
        LAYA_LAUNCH((few_dw_kernel<STEPS_T, false>), grid, block, 0, ctx->stream, p);
    check_launch("few_dw_kernel");
}

}  // namespace

void vocab_few_fwd(laya_ctx* ctx, const VocabArgs& a, float* row_loss, float* lse, float* loss, int* bad_count) {
    const int nb = blocks_of(a.rows), pitch = 16 * nb, steps = packed::steps_of(a.hidden);
    const int tiles = (a.vocab + FEW_V - 1) / FEW_V;
    unsigned* words;
    int* row_of;
    __bf16* x_rows;
    float2* part;
    carve(ctx, VOCAB_SLOT, [&](Carve& ws) {
        ws.take(words, WORDS);
        ws.take(row_of, a.rows);
        ws.take(x_rows, (size_t)steps * nb * 3 * FRAG);
        ws.take(part, (size_t)tiles * pitch);
    });
    const Prepare prep{a.x, a.row_weights, a.targets, a.rows, a.hidden, a.vocab, nb, x_rows, nullptr,
                       row_of, nullptr, bad_count, words, row_loss, lse};
    LAYA_LAUNCH(few_prepare_kernel, dim3(steps), dim3(256), 0, ctx->stream, prep);
    check_launch("few_prepare_kernel");
    FewLogits p{};
    p.W = a.W16 ? (const void*)a.W16 : (const void*)a.W;
    p.bias = a.bias;
    p.x_rows = x_rows;
    p.words = words;
    p.hidden = a.hidden;
    p.vocab = a.vocab;
    p.steps = steps;
    p.part = part;
    p.pitch = pitch;
    launch_logits<false>(ctx, a, p, nb);
    vocab_merge(ctx, a, part, pitch, tiles, words, row_of, row_loss, lse, loss);
}

void vocab_few_bwd(laya_ctx* ctx, const VocabArgs& a, const float* lse, float* dx, float* dW, float* db) {
    const int nb = blocks_of(a.rows), steps_t = (nb + 1) / 2, steps = packed::steps_of(a.hidden);
    const int tiles = (a.vocab + FEW_V - 1) / FEW_V, steps_v = packed::steps_of(a.vocab);
    // Slices of the vocabulary, so that few_dx's workgroups are about as many as the chip's CUs.
    const int across = (a.hidden + 255) / 256;
    const int per = std::max(4, (steps_v + std::max(1, ctx->cu_count / across) - 1) / std::max(1, ctx->cu_count / across));
    const int slices = (steps_v + per - 1) / per;
    unsigned* words;
    int *row_of, *place;
    __bf16 *x_rows, *x_cols, *g_rows, *g_cols;
    float* part;
    carve(ctx, VOCAB_SLOT, [&](Carve& ws) {
        ws.take(words, WORDS);
        ws.take(row_of, a.rows);
        ws.take(place, a.rows);
        ws.take(x_rows, (size_t)steps * nb * 3 * FRAG);
        ws.take(x_cols, (size_t)2 * steps * steps_t * 3 * FRAG);
        ws.take(g_rows, (size_t)tiles * (FEW_V / 32) * nb * 3 * FRAG);
        ws.take(g_cols, (size_t)tiles * (FEW_V / 16) * steps_t * 3 * FRAG);
        ws.take(part, (size_t)slices * 16 * nb * a.hidden);
    });
    const Prepare prep{a.x, a.row_weights, a.targets, a.rows, a.hidden, a.vocab, nb, x_rows, x_cols,
                       row_of, place, nullptr, words, nullptr, nullptr};
    LAYA_LAUNCH(few_prepare_kernel, dim3(steps), dim3(256), 0, ctx->stream, prep);
    check_launch("few_prepare_kernel");
    FewLogits p{};
    p.W = a.W16 ? (const void*)a.W16 : (const void*)a.W;
    p.bias = a.bias;
    p.x_rows = x_rows;
    p.words = words;
    p.hidden = a.hidden;
    p.vocab = a.vocab;
    p.steps = steps;
    p.row_of = row_of;
    p.targets = a.targets;
    p.lse = lse;
    p.weights = a.row_weights;
    p.g_rows = g_rows;
    p.g_cols = g_cols;
    p.db = db;
    p.scale = a.scale;
    launch_logits<true>(ctx, a, p, nb);
    if (dx) {
        const FewDx q{p.W, g_rows, a.hidden, a.vocab, steps_v, per, part};
        {
            ProfileScope scope(ctx, "vocab_few_dx", 2.0 * a.rows * a.hidden * a.vocab,
                               (a.W16 ? 2.0 : 4.0) * a.hidden * a.vocab);
            if (nb == 1) launch_dx<1>(ctx, a, q, slices);
            else if (nb == 2) launch_dx<2>(ctx, a, q, slices);
            else if (nb == 4) launch_dx<4>(ctx, a, q, slices);
            else launch_dx<8>(ctx, a, q, slices);
        }
        LAYA_LAUNCH(few_dx_sum_kernel, dim3((a.hidden + 255) / 256, a.rows), dim3(256), 0, ctx->stream, part, slices,
                    16 * nb, place, a.row_weights, a.scale, a.hidden, dx);
        check_launch("few_dx_sum_kernel");
    }
    if (dW) {
        const FewDw q{x_cols, g_cols, words, a.hidden, a.vocab, a.scale, dW};
        if (steps_t == 1) launch_dw<1>(ctx, a, q);
        else if (steps_t == 2) launch_dw<2>(ctx, a, q);
        else launch_dw<4>(ctx, a, q);
    }
}

}  // namespace laya
