// The vocabulary cross entropy of up to 256 rows, where the table's own bytes are the cost: every kernel reads W (or
// moves dW) once, straight from memory, and splits it in registers.
//
// The products are two-piece fp16 products (split.hpp) as the large ones, three matrix products each, but W is split as it
// streams by, so its scale is found on the way: a wave scales its 16 rows from the largest magnitude so far, with four
// bits to spare, and when a value would leave fp16's range it takes a new scale and brings its sums to it (a power of
// two, so exactly), as the running maximum of a softmax is handled. bf16 weights are one piece, two products.
//   few_prepare   the labelled rows' x as fragments, rows t over h and (weighted) rows h over t
//   few_logits    z = W·xᵀ, a wave 16 rows of W (its 8 k of a lane are two 16-byte loads); statistics, or G in both orders
//   few_dx        dxᵀ = Wᵀ·Gᵀ over slices of the vocabulary, a lane's 8 k eight loads down W's columns
//   few_dw        dWᵀ += xᵀ·G, a lane four neighbours of one row of dW
// Fragments are 16 rows x 32 k of v_mfma_f32_16x16x32_f16, [k / 8][row][8 k], the two planes one after another.
//
// A large copy runs at 5.0 TB/s on this card. 19 rows x 768 x 50368: logits 33.7 us (W's 155 MB at 4.6 TB/s); the merge and
// the preparation are 6 us of latency each. 77 rows both ways: logits 43 and 50 us, dx 47 us (3.3 TB/s: a lane's loads go
// down W's columns, eight bytes a row), dW 78 us (310 MB read and written, 4.0 TB/s). With more rows the splits and x's
// reads from LDS come to weigh as much: 192 rows 0.35 ms both ways, 256 rows 0.53 ms.
#include "elementwise.hpp"
#include "packed.hpp"
#include "vocab.hpp"

namespace laya {
namespace {

using packed::FRAG;
using packed::lds_byte;

constexpr int PLANES = 2, BLOCK = PLANES * FRAG;  // a fragment's fp16 values, both planes
constexpr int G_SCALE = 14;                       // |G| ≤ 1

__device__ __forceinline__ void split8(const float (&v)[8], float sc, f16x8 (&p)[2]) {
    f16x4 a[2], b[2];
    split2h_4(f32x4{v[0], v[1], v[2], v[3]}, sc, a[0], a[1]);
    split2h_4(f32x4{v[4], v[5], v[6], v[7]}, sc, b[0], b[1]);
#pragma unroll
    for (int k = 0; k < 2; ++k) p[k] = __builtin_shufflevector(a[k], b[k], 0, 1, 2, 3, 4, 5, 6, 7);
}
// c += a·b of two-piece operands (PA = 1: a is one piece), smallest products first.
template <int PA>
__device__ __forceinline__ void mma(const f16x8 (&a)[2], const f16x8 (&b)[2], f32x4& c) {
    if constexpr (PA == 2) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], b[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[0], c, 0, 0, 0);
}
__device__ __forceinline__ f16x8 fragment(const _Float16* at, int lane) {
    return *reinterpret_cast<const f16x8*>(at + lane * 8);
}

// The labelled rows in order, by every workgroup for itself: row_of[j] (LDS) and their number. VOCAB_FEW rows at most.
__device__ __forceinline__ int list_rows(const int* targets, int rows, int vocab, int* row_of, int& bad) {
    constexpr int WAVES = VOCAB_FEW / 64;
    __shared__ int wave_count[WAVES], wave_bad[WAVES];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int y = tid < rows ? targets[tid] : LAYA_NO_LABEL;
    const bool has = y >= 0 && y < vocab;
    const unsigned long long m = __ballot(has), wrong = __ballot(!has && y != LAYA_NO_LABEL);
    if (lane == 0 && wave < WAVES) {
        wave_count[wave] = __popcll(m);
        wave_bad[wave] = __popcll(wrong);
    }
    __syncthreads();
    int before = 0, count = 0;
    bad = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
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
    _Float16* x_rows;                   // [k step][block of t][2][FRAG], rows scaled by 2^exps[t]
    _Float16* x_cols;                   // [block of 16 h][step of 32 t][2][FRAG], weighted (null: not wanted)
    int* exps;
    int *row_of, *place, *bad_count;
    unsigned* words;
    float *row_loss, *lse;              // of the forward (null in the backward)
};

// One workgroup a step of 32 columns of x; each finds the rows' scales for itself.
__global__ __launch_bounds__(1024) void few_prepare_kernel(Prepare p) {
    __shared__ int row_of[VOCAB_FEW], row_exp[VOCAB_FEW];
    __shared__ float tile[VOCAB_FEW][33];
    __shared__ unsigned whole;
    const int tid = threadIdx.x, step = blockIdx.x;
    int bad;
    if (tid == 0) whole = 0;
    const int count = list_rows(p.targets, p.rows, p.vocab, row_of, bad);
    for (int j = tid >> 3; j < 16 * p.blocks_t; j += 128) {  // thread t four columns of row t / 8 of this step
        const int c = 32 * step + 4 * (tid & 7);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            tile[j][4 * (tid & 7) + i] =
                j < count && c + i < p.hidden ? p.x[(size_t)row_of[j] * p.hidden + c + i] : 0.0f;
    }
    for (int j = tid >> 4; j < 16 * p.blocks_t; j += 64) {  // 16 threads a row
        unsigned m = 0;
        if (j < count) {
            const float* row = p.x + (size_t)row_of[j] * p.hidden;
            int c = 4 * (tid & 15);
#pragma unroll 8
            for (; c + 4 <= p.hidden; c += 64) m = max(m, amax_bits4(*reinterpret_cast<const f32x4_any*>(row + c)));
            for (; c < p.hidden; ++c) m = max(m, amax_bits(row[c]));  // a piece of four
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
        if ((tid & 15) == 0) {
            const int e = pair_scale_exp(m);
            row_exp[j] = e;
            if (step == 0) p.exps[j] = e;
            if (j < count) {
                const float w = p.weights ? fabsf(p.weights[row_of[j]]) : 1.0f;
                atomicMax(&whole, amax_bits(__builtin_bit_cast(float, m) * w));
            }
        }
    }
    __syncthreads();
    if (step == 0) {
        if (tid < WORDS)
            p.words[tid] = tid == WORD_COUNT ? count : tid == WORD_BAD ? bad : tid == WORD_WX ? whole : 0;
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
    const int o = tid & 3, steps_t = (p.blocks_t + 1) / 2;
    float v[8];
    f16x8 f[2];
    for (int r = tid >> 2; r < 16 * p.blocks_t; r += 256) {  // row r over h, octet o
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = tile[r][8 * o + i];
        split8(v, exp2_int(row_exp[r]), f);
        _Float16* to = p.x_rows + ((size_t)step * p.blocks_t + (r >> 4)) * BLOCK + (o * 16 + (r & 15)) * 8;
#pragma unroll
        for (int k = 0; k < 2; ++k) *reinterpret_cast<f16x8*>(to + k * FRAG) = f[k];
    }
    if (!p.x_cols) return;
    for (int s = tid >> 7; s < steps_t; s += 8) {  // column 32·step + r over t, octet o of step s
        const int r = (tid >> 2) & 31;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = 32 * s + 8 * o + i;
            v[i] = t < count ? tile[t][r] * (p.weights ? p.weights[row_of[t]] : 1.0f) : 0.0f;
        }
        split8(v, exp2_int(pair_scale_exp(whole)), f);
        _Float16* to = p.x_cols + ((size_t)(2 * step + (r >> 4)) * steps_t + s) * BLOCK + (o * 16 + (r & 15)) * 8;
#pragma unroll
        for (int k = 0; k < 2; ++k) *reinterpret_cast<f16x8*>(to + k * FRAG) = f[k];
    }
}

// ------------------------------------------------------------------------------------------- shared

// Fragments that all waves of a workgroup read, copied to an LDS ring a step at a time: KB KB in a row a step, each of at
// least WAVES waves starting PER copies of 1 KB (some may repeat the last: the same bytes to the same place).
template <int KB, int WAVES, int RING>
struct Stream {
    static constexpr int PER = (KB + WAVES - 1) / WAVES, STEP = KB * FRAG;
    const _Float16* from;
    unsigned lds0;
    int chunk[PER], last;
    __device__ __forceinline__ Stream(const _Float16* data, const _Float16* lds, int wave, int lane, int steps)
        : from(data + lane * 8), lds0(lds_byte(lds)), last(steps - 1) {
#pragma unroll
        for (int k = 0; k < PER; ++k) chunk[k] = __builtin_amdgcn_readfirstlane(min(wave + k * (int)(blockDim.x >> 6), KB - 1));
    }
    // Step s into its slot; past the end the last step again, so that each step has as many copies under way.
    __device__ __forceinline__ void start(int s) const {
        const size_t at = (size_t)min(s, last) * STEP;
        const unsigned slot = lds0 + (unsigned)(s % RING) * (2 * STEP);
#pragma unroll
        for (int k = 0; k < PER; ++k) copy(at, slot, k);
    }
    // The same without the repeated copies, for who waits for all.
    __device__ __forceinline__ void start_once(int s, int wave) const {
        const size_t at = (size_t)s * STEP;
        const unsigned slot = lds0 + (unsigned)(s % RING) * (2 * STEP);
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (__builtin_amdgcn_readfirstlane(wave) + k * (int)(blockDim.x >> 6) < KB) copy(at, slot, k);
    }
    __device__ __forceinline__ void copy(size_t at, unsigned slot, int k) const {
        const unsigned to = slot + chunk[k] * (2 * FRAG);
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to),
                     "v"(from + at + chunk[k] * FRAG) : "memory");
    }
};

// Few-row products run in steps of 32 k with RING slots: step s starts the copies and the wave's own loads (LOADS of them,
// each an instruction) of step s + RING − 1. What a wave has started behind the copies of step s when it comes to it:
// the loads of steps s … s + RING − 2 and the copies of s + 1 … s + RING − 2. Waiting until no more than these are under
// way means that the copies have landed; memory accesses end in order.
template <int RING, int PER, int LOADS>
__device__ __forceinline__ void wait_step() {
    packed::wait_copies<(RING - 1) * LOADS + (RING - 2) * PER>();
}

// ------------------------------------------------------------------------------------------- logits

struct FewLogits {
    const void* W;
    const float* bias;
    const _Float16* x_rows;
    const int* exps;
    unsigned* words;
    int hidden, vocab, steps, blocks_v;  // blocks_v: blocks of 16 rows of W, an even number
    const int *row_of, *targets;
    // Statistics:
    float2* part;            // [workgroup][pitch]
    int pitch;
    float* z_target;         // [labelled row]: the target's logit as it is in the sum
    // G:
    const float *lse, *weights;
    _Float16* g_rows;        // [step of 32 v][block of t][2][FRAG]: rows t over v
    _Float16* g_cols;        // [block of 16 v][step of 32 t][2][FRAG]: rows v over t
    float* db;
    float scale;
};

// Blocks of 16 rows of W a wave takes: with many rows of x it is their reads from LDS that two blocks share.
constexpr int wave_blocks(int nb) { return nb >= 8 ? 2 : 1; }
// Steps of a ring: what is under way of W waits in registers. At 16 blocks the sums leave room for two (256 rows x 768 x
// 50368 both ways 527 us; with three, which spill more, 556).
constexpr int ring_of(int nb) { return nb >= 16 ? 2 : nb >= 12 ? 3 : 4; }

// A workgroup is as many waves, WAVES at least, as spread the table's blocks of 16 rows evenly over the CUs.
template <int NB, typename TW, bool GRAD, int WAVES>
__global__ __launch_bounds__(1024 / wave_blocks(NB), 1) void few_logits_kernel(FewLogits p) {
    constexpr int PW = sizeof(TW) == 2 ? 1 : 2, VB = wave_blocks(NB), RING = ring_of(NB);
    constexpr int LOADS = VB * (sizeof(TW) == 2 ? 1 : 2);
    typedef Stream<2 * NB, WAVES, RING> S;
    constexpr int PITCH = 36, ROOM = GRAD ? 16 * 16 * PITCH * 2 : 16 * 16 * NB * 4;  // what the end needs
    __shared__ __attribute__((aligned(16))) _Float16 lds[RING * S::STEP < ROOM ? ROOM : RING * S::STEP];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, waves = blockDim.x >> 6, steps = p.steps;
    const int v0 = (blockIdx.x * waves + wave) * (16 * VB);
    const TW* row[VB];
#pragma unroll
    for (int i = 0; i < VB; ++i)
        row[i] = static_cast<const TW*>(p.W) + (size_t)min(v0 + 16 * i + (lane & 15), p.vocab - 1) * p.hidden;
    const S x(p.x_rows, lds, wave, lane, steps);
    auto load = [&](int s, float (&w)[VB][8]) {
        const int c = min(32 * s + 8 * (lane >> 4), p.hidden - 8);  // the last 8 also for what reaches behind them
#pragma unroll
        for (int i = 0; i < VB; ++i) load8(row[i] + c, w[i]);
    };
    float w[RING][VB][8];
    int e = 126;           // of the wave's scale
    float limit = 0.0f;    // magnitudes from here on need another
    float top = 0.0f;      // the lane's largest
    f32x4 acc[VB][NB];
#pragma unroll
    for (int i = 0; i < VB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{};
#pragma unroll
    for (int k = 0; k < RING - 1; ++k) {
        x.start(k);
        load(k, w[k]);
    }
    auto step = [&](int s, auto slot) {
        constexpr int K = decltype(slot)::value;
        // Step s's copies have landed for every wave, and step s − 1 is read by all: its slot is free.
        wait_step<RING, S::PER, LOADS>();
        x.start(s + RING - 1);
        load(s + RING - 1, w[(K + RING - 1) % RING]);
        __builtin_amdgcn_sched_barrier(0);  // not to the step's end, where the scheduler would have them
        if (32 * s + 32 > p.hidden) {  // the last step: what was loaded from the row's end moves to its place
            const int left = p.hidden - 32 * s - 8 * (lane >> 4);
            for (int q = p.hidden & 7; q > 0 && q < 8; ++q)
#pragma unroll
                for (int i = 0; i < VB; ++i)
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (left > 0 && left < 8) w[K][i][k] = k < 7 ? w[K][i][k + 1 < 8 ? k + 1 : 7] : 0.0f;
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) w[K][i][k] = left > 0 ? w[K][i][k] : 0.0f;
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < VB; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(w[K][i][k]));
        if (__any(m >= limit)) {  // a new scale (of infinities, none: they reach the sums as such)
            unsigned bits = 0;
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) bits = max(bits, amax_bits(w[K][i][k]));
            m = __builtin_bit_cast(float, bits);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) bits = max(bits, (unsigned)__shfl_xor((int)bits, o, 64));
            const int to = min(e, pair_scale_exp(bits) - 3);
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_amdgcn_ldexpf(acc[i][j][r], to - e);
            e = to;
            limit = exp2_int(min(15 - e, 127));
        }
        if (GRAD) top = fmaxf(top, m);
        f16x8 a[VB][2];
#pragma unroll
        for (int i = 0; i < VB; ++i) split8(w[K][i], exp2_int(max(e, -126)), a[i]);
        const _Float16* xs = lds + K * S::STEP;
        // A block of x ahead, and no more (the scheduler would hold them all).
        f16x8 b[2][2];
#pragma unroll
        for (int q = 0; q < 2; ++q) b[0][q] = fragment(xs + q * FRAG, lane);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            if (j + 1 < NB)
#pragma unroll
                for (int q = 0; q < 2; ++q) b[(j + 1) & 1][q] = fragment(xs + (2 * (j + 1) + q) * FRAG, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < VB; ++i) mma<PW>(a[i], b[j & 1], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int s = 0; s < steps; s += RING) {
        step(s, std::integral_constant<int, 0>());
        if (s + 1 < steps) step(s + 1, std::integral_constant<int, 1>());
        if constexpr (RING > 2)
            if (s + 2 < steps) step(s + 2, std::integral_constant<int, 2>());
        if constexpr (RING == 4)
            if (s + 3 < steps) step(s + 3, std::integral_constant<int, 3>());
    }
    packed::wait_copies<0>();
    const int count = (int)p.words[WORD_COUNT];
#pragma unroll
    for (int i = 0; i < VB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int v = v0 + 16 * i + 4 * (lane >> 4) + r;
            const float b = v < p.vocab ? (p.bias ? p.bias[v] : 0.0f) : -__builtin_inff();
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[i][j][r] = __builtin_amdgcn_ldexpf(acc[i][j][r], -(e + p.exps[16 * j + (lane & 15)])) + b;
        }
    if constexpr (!GRAD) {
        if (v0 < p.blocks_v * 16) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int t = 16 * j + (lane & 15);
                const int where = (t < count ? p.targets[p.row_of[t]] : -1) - (v0 + 4 * (lane >> 4));
                if (!__any(where >= 0 && where < 16 * VB)) continue;
#pragma unroll
                for (int i = 0; i < VB; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (where == 16 * i + r) p.z_target[t] = acc[i][j][r];
            }
        }
        float2* red = reinterpret_cast<float2*>(lds);  // [wave][16·NB]
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float m = -__builtin_inff(), s = 0.0f;
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[i][j][r]);
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float at = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < VB; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[i][j][r] - at) * LOG2E);
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            if (lane < 16) red[wave * (16 * NB) + 16 * j + lane] = make_float2(m, s);
        }
        __syncthreads();
        for (int t = tid; t < 16 * NB; t += blockDim.x) {
            float m = -__builtin_inff(), s = 0.0f;
            for (int q = 0; q < waves; ++q) m = fmaxf(m, red[q * (16 * NB) + t].x);
            const float at = m == -__builtin_inff() ? 0.0f : m;
            for (int q = 0; q < waves; ++q) {
                const float2 a = red[q * (16 * NB) + t];
                s += a.y * __builtin_amdgcn_exp2f((a.x - at) * LOG2E);
            }
            p.part[(size_t)blockIdx.x * p.pitch + t] = make_float2(m, s);
        }
    } else {
        __shared__ unsigned largest;
        if (tid == 0) largest = 0;
        __syncthreads();
        atomicMax(&largest, __builtin_bit_cast(unsigned, top));
        __syncthreads();
        if (tid == 0) atomicMax(p.words + WORD_W, largest);
        if (v0 >= p.blocks_v * 16) return;
        constexpr int STEPS_T = (NB + 1) / 2;
        float* turn = reinterpret_cast<float*>(lds) + wave * (16 * PITCH);
#pragma unroll
        for (int i = 0; i < VB; ++i) {
            const int vb = v0 + 16 * i;
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
                        const int y = (live ? p.targets[r] : -1) - (vb + 4 * (lane >> 4));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float q = __builtin_amdgcn_exp2f((acc[i][j][e] - lse) * LOG2E);
                            q -= y == e ? 1.0f : 0.0f;
                            g[e] = live ? q * (float)(1 << G_SCALE) : 0.0f;
                        }
                        const float wt = live ? (p.weights ? p.weights[r] : 1.0f) : 0.0f;
                        db += live ? g * wt : f32x4{};
                        f16x4 f[2];
                        split2h_4(g, 1.0f, f[0], f[1]);
                        _Float16* to = p.g_rows + ((size_t)(vb >> 5) * NB + j) * BLOCK +
                                     ((((vb >> 4) & 1) * 2 + (lane >> 5)) * 16 + (lane & 15)) * 8 + 4 * ((lane >> 4) & 1);
#pragma unroll
                        for (int q = 0; q < 2; ++q) *reinterpret_cast<f16x4*>(to + q * FRAG) = f[q];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) turn[(4 * (lane >> 4) + e) * PITCH + 16 * jj + (lane & 15)] = g[e];
                }
                float v[8];
                f16x8 f[2];
                const float* at = turn + (lane & 15) * PITCH + 8 * (lane >> 4);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = at[e];
                split8(v, 1.0f, f);
                _Float16* to = p.g_cols + ((size_t)(vb >> 4) * STEPS_T + ts) * BLOCK + lane * 8;
#pragma unroll
                for (int q = 0; q < 2; ++q) *reinterpret_cast<f16x8*>(to + q * FRAG) = f[q];
            }
            if (p.db) {
#pragma unroll
                for (int o = 1; o < 16; o <<= 1)
#pragma unroll
                    for (int e = 0; e < 4; ++e) db[e] += __shfl_xor(db[e], o, 64);
                const int v = vb + 4 * (lane >> 4);
                if ((lane & 15) == 0)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (v + e < p.vocab) p.db[v + e] += db[e] * (1.0f / (1 << G_SCALE)) * p.scale;
            }
        }
    }
}

// -------------------------------------------------------------------------------------------- dx

struct FewDx {
    const void* W;
    const _Float16* g_rows;
    const unsigned* words;
    int hidden, vocab, steps, per;  // steps of 32 v in all, and of a slice
    float* part;                    // [slice][16·NB][hidden]
};

// A workgroup: 256 columns of W over a slice of the vocabulary; a wave 32 of them, block i the columns 2·n + i, so that a
// lane's two blocks come with one load a row.
template <int NB, typename TW>
__global__ __launch_bounds__(512, 1) void few_dx_kernel(FewDx p) {
    constexpr int PW = sizeof(TW) == 2 ? 1 : 2, LOADS = 8, RING = 4;
    typedef Stream<2 * NB, 8, RING> S;
    __shared__ __attribute__((aligned(16))) _Float16 lds[RING * S::STEP];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = blockIdx.y * p.per, steps = min(p.per, p.steps - first);
    const int h0 = blockIdx.x * 256 + wave * 32;
    const TW* W = static_cast<const TW*>(p.W);
    const S g(p.g_rows + (size_t)first * S::STEP, lds, wave, lane, steps);
    // The last pair for what reaches behind it; of an odd width its second is the last column.
    const int col = min(h0 + 2 * (lane & 15), p.hidden - 2);
    const bool second = h0 + 2 * (lane & 15) == p.hidden - 1;
    // Rows behind the vocabulary read its last: G is zero there.
    auto load = [&](int s, float (&w)[2][8]) {
        const int v = 32 * (first + min(s, steps - 1)) + 8 * (lane >> 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const TW* at = W + (size_t)min(v + e, p.vocab - 1) * p.hidden;
            typedef TW Pair __attribute__((ext_vector_type(2), aligned(sizeof(TW))));
            const Pair both = *reinterpret_cast<const Pair*>(at + col);
            w[0][e] = (float)both[0];
            w[1][e] = (float)both[1];
        }
    };
    const int ew = pair_scale_exp(p.words[WORD_W]);
    const float sc = exp2_int(ew);
    float w[RING][2][8];
    f32x4 acc[2][NB];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{};
#pragma unroll
    for (int k = 0; k < RING - 1; ++k) {
        g.start(k);
        load(k, w[k]);
    }
    auto step = [&](int s, auto slot) {
        constexpr int K = decltype(slot)::value;
        wait_step<RING, S::PER, LOADS>();
        g.start(s + RING - 1);
        load(s + RING - 1, w[(K + RING - 1) % RING]);
        __builtin_amdgcn_sched_barrier(0);  // not to the step's end, where the scheduler would have them
        f16x8 a[2][2], b[2][2];
        if (second)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[K][0][e] = w[K][1][e];
        split8(w[K][0], sc, a[0]);
        split8(w[K][1], sc, a[1]);
        const _Float16* gs = lds + K * S::STEP;
#pragma unroll
        for (int q = 0; q < 2; ++q) b[0][q] = fragment(gs + q * FRAG, lane);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            if (j + 1 < NB)
#pragma unroll
                for (int q = 0; q < 2; ++q) b[(j + 1) & 1][q] = fragment(gs + (2 * (j + 1) + q) * FRAG, lane);
            __builtin_amdgcn_sched_barrier(0);
            mma<PW>(a[0], b[j & 1], acc[0][j]);
            mma<PW>(a[1], b[j & 1], acc[1][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int s = 0; s < steps; s += RING) {
        step(s, std::integral_constant<int, 0>());
        if (s + 1 < steps) step(s + 1, std::integral_constant<int, 1>());
        if (s + 2 < steps) step(s + 2, std::integral_constant<int, 2>());
        if constexpr (RING == 4)
            if (s + 3 < steps) step(s + 3, std::integral_constant<int, 3>());
    }
    packed::wait_copies<0>();
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        float* to = p.part + ((size_t)blockIdx.y * (16 * NB) + 16 * j + (lane & 15)) * p.hidden;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int h = h0 + 2 * (4 * (lane >> 4) + e) + i;
                if (h < p.hidden) to[h] = __builtin_amdgcn_ldexpf(acc[i][j][e], -(G_SCALE + ew));
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
#pragma unroll 4
        for (; k + 3 < slices; k += 4)
#pragma unroll
            for (int q = 0; q < 4; ++q) s[q] += at[(k + q) * next];
        for (; k < slices; ++k) s[0] += at[k * next];
    }
    dx[(size_t)r * hidden + h] = j >= 0 ? ((s[0] + s[1]) + (s[2] + s[3])) * (weights ? weights[r] : 1.0f) * scale : 0.0f;
}

// -------------------------------------------------------------------------------------------- dW

struct FewDw {
    const _Float16 *x_cols, *g_cols;
    const unsigned* words;
    int hidden, vocab, blocks_v;
    float scale;
    float* dW;
};

// A wave: 16 rows of dW, their G in registers, HB blocks of 16 columns at a time. A chunk's x comes through LDS, its dW to
// registers, both started while the chunk before is computed.
template <int STEPS_T>
__global__ __launch_bounds__(1024, 1) void few_dw_kernel(FewDw p) {
    if (p.words[WORD_COUNT] == 0) return;
    constexpr int HB = STEPS_T == 1 ? 8 : STEPS_T <= 4 ? 4 : 2;
    typedef Stream<2 * STEPS_T * HB, 4, 2> S;
    __shared__ __attribute__((aligned(16))) _Float16 lds[2 * S::STEP];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, vb = blockIdx.x * (int)(blockDim.x >> 6) + wave;
    const int v = 16 * vb + (lane & 15), chunks = (p.hidden + 16 * HB - 1) / (16 * HB);
    const bool live = v < p.vocab;
    const int e = -(G_SCALE + pair_scale_exp(p.words[WORD_WX]));
    f16x8 g[STEPS_T][2];
#pragma unroll
    for (int s = 0; s < STEPS_T; ++s)
#pragma unroll
        for (int q = 0; q < 2; ++q)
            g[s][q] = fragment(p.g_cols + (((size_t)min(vb, p.blocks_v - 1) * STEPS_T + s) * 2 + q) * FRAG, lane);
    float* row = p.dW + (size_t)min(v, p.vocab - 1) * p.hidden;
    const S x(p.x_cols, lds, wave, lane, chunks);
    auto fetch = [&](int chunk, int k) {
        const int h = 16 * (chunk * HB + k) + 4 * (lane >> 4);
        f32x4 o = {};
        if (h + 4 <= p.hidden) {
            o = *reinterpret_cast<const f32x4_any*>(row + h);
        } else if (h < p.hidden) {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (h + e < p.hidden) o[e] = row[h + e];
        }
        return o;
    };
    f32x4 next[HB];
    x.start_once(0, wave);
#pragma unroll
    for (int k = 0; k < HB; ++k) next[k] = fetch(0, k);
    for (int c = 0; c < chunks; ++c) {
        packed::wait_copies<0>();
        f32x4 now[HB];
#pragma unroll
        for (int k = 0; k < HB; ++k) now[k] = next[k];
        if (c + 1 < chunks) {
            x.start_once(c + 1, wave);
#pragma unroll
            for (int k = 0; k < HB; ++k) next[k] = fetch(c + 1, k);
        }
        const _Float16* xs = lds + (c & 1) * S::STEP;
#pragma unroll
        for (int k = 0; k < HB; ++k) {
            f32x4 sum = {};
#pragma unroll
            for (int s = 0; s < STEPS_T; ++s) {
                f16x8 a[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) a[q] = fragment(xs + ((k * STEPS_T + s) * 2 + q) * FRAG, lane);
                mma<2>(a, g[s], sum);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) now[k][r] += __builtin_amdgcn_ldexpf(sum[r], e) * p.scale;
            const int h = 16 * (c * HB + k) + 4 * (lane >> 4);
            if (!live) continue;
            if (h + 4 <= p.hidden) {
                *reinterpret_cast<f32x4_any*>(row + h) = now[k];
            } else if (h < p.hidden) {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (h + e < p.hidden) row[h + e] = now[k][e];
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ launches

int blocks_of(const VocabArgs& a) {
    const int b = (a.rows + 15) / 16;
    return b <= 6 ? b : b <= 8 ? 8 : b <= 10 ? 10 : b <= 12 ? 12 : 16;
}

// Waves of a workgroup that takes `each` blocks of 16 rows of W a wave: as few as take the table in the rounds that 16
// blocks a workgroup would take, one workgroup a CU, and 4 at least.
int waves_of(const laya_ctx* ctx, int blocks_v, int each = 1) {
    const int rounds = (blocks_v + 16 * ctx->cu_count - 1) / (16 * ctx->cu_count);
    const int units = (blocks_v + each - 1) / each;
    return std::max(4, (units + rounds * ctx->cu_count - 1) / (rounds * ctx->cu_count));
}

// f(the number of blocks as a constant).
template <class F> void with_blocks(int nb, F&& f) {
    if (nb == 1) f(std::integral_constant<int, 1>());
    else if (nb == 2) f(std::integral_constant<int, 2>());
    else if (nb == 3) f(std::integral_constant<int, 3>());
    else if (nb == 4) f(std::integral_constant<int, 4>());
    else if (nb == 5) f(std::integral_constant<int, 5>());
    else if (nb == 6) f(std::integral_constant<int, 6>());
    else if (nb == 8) f(std::integral_constant<int, 8>());
    else if (nb == 10) f(std::integral_constant<int, 10>());
    else if (nb == 12) f(std::integral_constant<int, 12>());
    else f(std::integral_constant<int, 16>());
}

void launch_prepare(laya_ctx* ctx, const Prepare& p, int steps) {
    LAYA_LAUNCH(few_prepare_kernel, dim3(steps), dim3(1024), 0, ctx->stream, p);
    check_launch("few_prepare_kernel");
}

template <bool GRAD>
void launch_logits(laya_ctx* ctx, const VocabArgs& a, const FewLogits& p, int nb) {
    const int each = wave_blocks(nb), waves = waves_of(ctx, p.blocks_v, each);
    const dim3 grid((p.blocks_v + waves * each - 1) / (waves * each)), block(64 * waves);
    ProfileScope scope(ctx, "vocab_few_logits", 2.0 * a.rows * a.hidden * a.vocab,
                       (a.W16 ? 2.0 : 4.0) * a.hidden * a.vocab);
    with_blocks(nb, [&](auto n) {
        constexpr int NB = decltype(n)::value;
        constexpr int MANY = wave_blocks(NB) == 2 ? 6 : 8;
        if (a.W16 && waves >= MANY)
            LAYA_LAUNCH((few_logits_kernel<NB, __bf16, GRAD, MANY>), grid, block, 0, ctx->stream, p);
        else if (a.W16)
            LAYA_LAUNCH((few_logits_kernel<NB, __bf16, GRAD, 4>), grid, block, 0, ctx->stream, p);
        else if (waves >= MANY)
            LAYA_LAUNCH((few_logits_kernel<NB, float, GRAD, MANY>), grid, block, 0, ctx->stream, p);
        else
            LAYA_LAUNCH((few_logits_kernel<NB, float, GRAD, 4>), grid, block, 0, ctx->stream, p);
    });
    check_launch("few_logits_kernel");
}

void launch_dx(laya_ctx* ctx, const VocabArgs& a, const FewDx& p, int slices, int nb) {
    const dim3 grid((a.hidden + 255) / 256, slices), block(512);
    ProfileScope scope(ctx, "vocab_few_dx", 2.0 * a.rows * a.hidden * a.vocab,
                       (a.W16 ? 2.0 : 4.0) * a.hidden * a.vocab);
    with_blocks(nb, [&](auto n) {
        constexpr int NB = decltype(n)::value;
        if (a.W16)
            LAYA_LAUNCH((few_dx_kernel<NB, __bf16>), grid, block, 0, ctx->stream, p);
        else
            LAYA_LAUNCH((few_dx_kernel<NB, float>), grid, block, 0, ctx->stream, p);
    });
    check_launch("few_dx_kernel");
}

template <int STEPS_T>
void launch_dw(laya_ctx* ctx, const VocabArgs& a, const FewDw& p, int waves) {
    const dim3 grid((p.blocks_v + waves - 1) / waves), block(64 * waves);
    ProfileScope scope(ctx, "vocab_few_dw", 2.0 * a.rows * a.hidden * a.vocab, 8.0 * a.hidden * a.vocab);
    LAYA_LAUNCH(few_dw_kernel<STEPS_T>, grid, block, 0, ctx->stream, p);
    check_launch("few_dw_kernel");
}

}  // namespace

bool vocab_few_rows(const VocabArgs& a) { return a.rows <= VOCAB_FEW && a.hidden >= 8; }  // rows of whole octets

void vocab_few_fwd(laya_ctx* ctx, const VocabArgs& a, float* row_loss, float* lse, float* loss, int* bad_count) {
    const int nb = blocks_of(a), pitch = 16 * nb, steps = packed::steps_of(a.hidden);
    const int blocks_v = 2 * packed::steps_of(a.vocab), rows_of_wg = wave_blocks(nb) * waves_of(ctx, blocks_v, wave_blocks(nb));
    const int tiles = (blocks_v + rows_of_wg - 1) / rows_of_wg;
    unsigned* words;
    int* row_of;
    _Float16* x_rows;
    int* exps;
    float2* part;
    float* z_target;
    carve(ctx, VOCAB_SLOT, [&](Carve& ws) {
        ws.take(words, WORDS);
        ws.take(row_of, a.rows);
        ws.take(exps, 16 * nb);
        ws.take(x_rows, (size_t)steps * nb * BLOCK);
        ws.take(part, (size_t)tiles * pitch);
        ws.take(z_target, pitch);
    });
    const Prepare prep{a.x, a.row_weights, a.targets, a.rows, a.hidden, a.vocab, nb, x_rows, nullptr, exps,
                       row_of, nullptr, bad_count, words, row_loss, lse};
    launch_prepare(ctx, prep, steps);
    FewLogits p{};
    p.W = a.W16 ? (const void*)a.W16 : (const void*)a.W;
    p.bias = a.bias;
    p.x_rows = x_rows;
    p.exps = exps;
    p.words = words;
    p.hidden = a.hidden;
    p.vocab = a.vocab;
    p.steps = steps;
    p.blocks_v = blocks_v;
    p.row_of = row_of;
    p.targets = a.targets;
    p.part = part;
    p.z_target = z_target;
    p.pitch = pitch;
    launch_logits<false>(ctx, a, p, nb);
    vocab_merge(ctx, a, part, pitch, tiles, words, row_of, z_target, row_loss, lse, loss);
}

void vocab_few_bwd(laya_ctx* ctx, const VocabArgs& a, const float* lse, float* dx, float* dW, float* db) {
    const int nb = blocks_of(a), steps_t = (nb + 1) / 2, steps = packed::steps_of(a.hidden);
    const int steps_v = packed::steps_of(a.vocab), blocks_v = 2 * steps_v, waves = waves_of(ctx, blocks_v);
    // Slices of the vocabulary, so that few_dx's workgroups are about as many as the chip's CUs.
    const int across = (a.hidden + 255) / 256;
    const int per = std::max(4, (steps_v + std::max(1, ctx->cu_count / across) - 1) / std::max(1, ctx->cu_count / across));
    const int slices = (steps_v + per - 1) / per;
    unsigned* words;
    int *row_of, *place;
    _Float16 *x_rows, *x_cols, *g_rows, *g_cols;
    int* exps;
    float* part;
    carve(ctx, VOCAB_SLOT, [&](Carve& ws) {
        ws.take(words, WORDS);
        ws.take(row_of, a.rows);
        ws.take(place, a.rows);
        ws.take(exps, 16 * nb);
        ws.take(x_rows, (size_t)steps * nb * BLOCK);
        ws.take(x_cols, (size_t)(2 * steps + 6) * steps_t * BLOCK);  // few_dw reads whole chunks of up to 8 blocks
        ws.take(g_rows, (size_t)steps_v * nb * BLOCK);
        ws.take(g_cols, (size_t)blocks_v * steps_t * BLOCK);
        ws.take(part, (size_t)slices * 16 * nb * a.hidden);
    });
    const Prepare prep{a.x, a.row_weights, a.targets, a.rows, a.hidden, a.vocab, nb, x_rows, x_cols, exps,
                       row_of, place, nullptr, words, nullptr, nullptr};
    launch_prepare(ctx, prep, steps);
    FewLogits p{};
    p.W = a.W16 ? (const void*)a.W16 : (const void*)a.W;
    p.bias = a.bias;
    p.x_rows = x_rows;
    p.exps = exps;
    p.words = words;
    p.hidden = a.hidden;
    p.vocab = a.vocab;
    p.steps = steps;
    p.blocks_v = blocks_v;
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
        const FewDx q{p.W, g_rows, words, a.hidden, a.vocab, steps_v, per, part};
        launch_dx(ctx, a, q, slices, nb);
        LAYA_LAUNCH(few_dx_sum_kernel, dim3((a.hidden + 255) / 256, a.rows), dim3(256), 0, ctx->stream, part, slices,
                    16 * nb, place, a.row_weights, a.scale, a.hidden, dx);
        check_launch("few_dx_sum_kernel");
    }
    if (dW) {
        const FewDw q{x_cols, g_cols, words, a.hidden, a.vocab, blocks_v, a.scale, dW};
        if (steps_t == 1) launch_dw<1>(ctx, a, q, waves);
        else if (steps_t == 2) launch_dw<2>(ctx, a, q, waves);
        else if (steps_t == 3) launch_dw<3>(ctx, a, q, waves);
        else if (steps_t == 4) launch_dw<4>(ctx, a, q, waves);
        else if (steps_t == 5) launch_dw<5>(ctx, a, q, waves);
        else if (steps_t == 6) launch_dw<6>(ctx, a, q, waves);
        else launch_dw<8>(ctx, a, q, waves);
    }
}

}  // namespace laya
