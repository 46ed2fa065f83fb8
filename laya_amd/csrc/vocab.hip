// Softmax cross entropy of hidden states over a vocabulary, with its gradient, in pieces of the vocabulary.
//
//   z_tv = W_v·x_t + b_v,   L_t = log Σ_v exp z_tv − z_t,y_t,   loss = Σ_t w_t·L_t
//   G_tv = exp(z_tv − lse_t) − [v = y_t],   dx_t = w_t·Σ_v G_tv·W_v,   dW_v += Σ_t G_tv·(w_t·x_t),   db_v += Σ_t w_t·G_tv
//
// The logits are never kept: the forward reduces each tile of them to a maximum and a sum of exponentials a row, merged
// at the end; the backward computes a piece's logits again and keeps its G as packed fp16 pieces (packed.hpp) just long
// enough for the piece's two products. Rows without a label are dropped first (label_rows), so that a batch with labels
// on 15 % of its tokens costs the products of those alone.
//
// Scales of the two-piece products (powers of two, so that scaling is exact): x by row, G by 2^14, w_t·x_t as a whole. W
// by row in the forward; as a whole in the backward, where one packed W serves the logits (over its columns) and dx
// (over its rows), as one packed G serves dx and dW.
//
// The matrix cores bound it, at the clock that their power leaves: a large fp16 library product of random values reaches
// 1.46 PFLOP/s on this card, 487 TFLOP/s of three products each. 4915 labelled rows x 768 x 50368: statistics 0.95 ms (399
// TFLOP/s of fp32 products), G 1.05 ms (362; it also writes 1 GB of pieces), the two gradient products 1.89 ms (403). What
// remains is copies: packing W 64 us (310 MB, 4.8 TB/s) in either direction, its largest magnitude 41 us (155 MB). Packing
// first pays because a tile's operands are read by every tile of their row and column: pieces are copied to LDS as they
// are, without a split in the product's loop.
#include "elementwise.hpp"
#include "packed.hpp"
#include "vocab.hpp"

namespace laya {
namespace {

using namespace packed;

constexpr int TILE = 256;            // what rows are padded to: the larger of the products' tiles
constexpr int G_SCALE = 14;          // |G| ≤ 1
constexpr int MAX_SPLITS = 32;       // ways of dx's sum over a piece of the vocabulary, and of dW's over the rows
constexpr size_t PIECE_BYTES = (size_t)3 << 30;  // of packed table and G that a piece of the vocabulary may take

// Square tiles of the products and how many workgroups share a CU.
template <int SIZE_, int WAVES_N, int PER_CU_>
struct Config {
    static constexpr int SIZE = SIZE_, WN = WAVES_N, PER_CU = PER_CU_, BM = SIZE / 32, BN = SIZE / 16 / WN;
    static constexpr int THREADS = 128 * WN, WM_ROWS = SIZE / 2, WN_COLS = SIZE / WN;
    template <int PA, int PB, bool TA = false, bool TB = false>
    using Tile = packed::Tile<2, WN, BM, BN, PA, PB, TA, TB, 2>;
};
typedef Config<256, 4, 1> T256;
typedef Config<128, 2, 2> T128;

// ------------------------------------------------------------------------------------------- labels

// One workgroup lists the labelled rows in order: row_of[j] for j < count, place[r] = j or −1. A target of
// LAYA_NO_LABEL carries no label; any other outside [0, vocab) is counted and carries none either. Bound by the latency of
// a round's loads and barriers: eight rows a thread at a time (13871 rows: 11 us, 18 with one).
__global__ __launch_bounds__(1024) void label_rows_kernel(const int* __restrict__ targets, int rows, int vocab,
                                                          int* __restrict__ row_of, int* __restrict__ place,
                                                          unsigned* words, int* bad_count, float* row_loss,
                                                          float* lse) {
    constexpr int EACH = 8;
    __shared__ int wave_count[EACH][16], wave_bad[16];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    int base = 0, wrong = 0;
    for (int r0 = 0; r0 < rows; r0 += EACH * 1024) {
        int at[EACH];
        bool has[EACH];
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int r = r0 + k * 1024 + tid;
            at[k] = r < rows ? targets[r] : LAYA_NO_LABEL;
        }
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            has[k] = at[k] >= 0 && at[k] < vocab;
            wrong += !has[k] && at[k] != LAYA_NO_LABEL ? 1 : 0;
            const unsigned long long m = __ballot(has[k]);
            at[k] = __popcll(m & ((1ull << lane) - 1));
            if (lane == 0) wave_count[k][wave] = __popcll(m);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const int r = r0 + k * 1024 + tid;
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                if (w < wave) at[k] += wave_count[k][w];
            }
            at[k] += base;
#pragma unroll
            for (int w = 0; w < 16; ++w) base += wave_count[k][w];
            if (has[k]) row_of[at[k]] = r;
            if (r < rows) {
                if (place) place[r] = has[k] ? at[k] : -1;
                if (!has[k] && row_loss) {
                    row_loss[r] = 0.0f;
                    lse[r] = 0.0f;
                }
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) wrong += __shfl_xor(wrong, o, 64);
    if (lane == 0) wave_bad[wave] = wrong;
    __syncthreads();
    int bad = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) bad += wave_bad[w];
    if (tid < WORDS) words[tid] = tid == WORD_COUNT ? base : tid == WORD_BAD ? bad : 0;
    if (tid == 0 && bad_count) *bad_count = bad;
}

// ------------------------------------------------------------------------------------------ packing

struct PackRows {
    const void* src;         // [.., K]
    const int* row_of;       // source row of packed row j (null: j itself)
    const unsigned* count;   // rows on the device (null: `rows`)
    int rows, K;
    const unsigned* whole;   // bits of the operand's largest magnitude, its scale (null: each row has its own)
    int* exps;               // [rows padded to TILE]: the exponent of each row's scale
    _Float16* out;
    const float* bias;       // with `padded`: bias (or zeros) by row, −∞ behind the last
    float* padded;
    const float* weights;    // of the gathered source rows (null: 1), for `wx`
    unsigned* wx;            // max |weight·x| as bits (null: not wanted)
};

// One workgroup packs 32 rows, scaled so that the largest finite magnitude (a row's own, or the operand's) lies in
// [2^14, 2^15). Row scales take one read for the magnitudes and one, from the caches, for the pieces. Thread t holds 8
// columns of row t / 8. T: fp32 or bf16 source.
template <typename T, int PLANES>
__global__ __launch_bounds__(256) void pack_rows_kernel(PackRows p) {
    const int b = blockIdx.x, tid = threadIdx.x, r = tid >> 3, o = tid & 7;
    const int rows = p.count ? (int)*p.count : p.rows;
    const int j = 32 * b + r;
    if (32 * b >= rows) {  // behind the last group: what the tiles that reach over it read by row
        if (o == 0 && p.padded) {
            p.exps[j] = 0;
            p.padded[j] = -__builtin_inff();
        }
        return;
    }
    const bool live = j < rows;
    const int from = live ? (p.row_of ? p.row_of[j] : j) : 0;
    const T* row = static_cast<const T*>(p.src) + (size_t)from * p.K;
    unsigned am = 0;
    if (p.whole) {
        am = *p.whole;
    } else {
        if (live)
            for (int c = o * 8; c < p.K; c += 64) {
                float v[8];
                load8(row, c, p.K, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) am = max(am, amax_bits(v[i]));
            }
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) am = max(am, (unsigned)__shfl_xor((int)am, s, 64));
    }
    const int e = pair_scale_exp(am);
    if (o == 0) {
        if (p.exps) p.exps[j] = live ? e : 0;
        if (p.padded) p.padded[j] = live ? (p.bias ? p.bias[j] : 0.0f) : -__builtin_inff();
    }
    if (p.wx) {
        const float w = live && p.weights ? fabsf(p.weights[from]) : 1.0f;
        unsigned m = live ? amax_bits(__builtin_bit_cast(float, am) * w) : 0u;
#pragma unroll
        for (int s = 8; s < 64; s <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, s, 64));
        if ((tid & 63) == 0 && m) atomicMax(p.wx, m);
    }
    const float sc = exp2_int(e);
    const int steps = (p.K + 31) / 32;
    for (int c = o * 8; c < steps * 32; c += 64) {
        float v[8] = {};
        if (live) load8(row, c, p.K, v);
        f16x8 hi, lo;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            _Float16 h, l;
            split_value(v[i] * sc, h, l);
            hi[i] = h;
            lo[i] = l;
        }
        _Float16* at = p.out + ((size_t)b * steps + (c >> 5)) * (2 * PLANES * FRAG) + unit_at<PLANES>(r, o & 3);
        *reinterpret_cast<f16x8*>(at) = hi;
        if constexpr (PLANES == 2) *reinterpret_cast<f16x8*>(at + FRAG) = lo;
    }
}

// max |x| over the finite values, as bits folded into *word.
template <typename T>
__global__ __launch_bounds__(256) void table_amax_kernel(const T* __restrict__ x, size_t n, unsigned* word) {
    constexpr int V = 16 / sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    unsigned m = 0;
    const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x, all = (size_t)gridDim.x * 256;
    const size_t nv = n / V;
    const Vec* xv = reinterpret_cast<const Vec*>(x);
    size_t i = at;
    for (; i + 3 * all < nv; i += 4 * all) {
        const Vec a = xv[i], b = xv[i + all], c = xv[i + 2 * all], d = xv[i + 3 * all];
#pragma unroll
        for (int k = 0; k < V; ++k)
            m = max(m, max(max(amax_bits((float)a[k]), amax_bits((float)b[k])),
                           max(amax_bits((float)c[k]), amax_bits((float)d[k]))));
    }
    for (; i < nv; i += all) {
        const Vec a = xv[i];
#pragma unroll
        for (int k = 0; k < V; ++k) m = max(m, amax_bits((float)a[k]));
    }
    for (i = nv * V + at; i < n; i += all) m = max(m, amax_bits((float)x[i]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
    __shared__ unsigned red[4];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        m = max(max(red[0], red[1]), max(red[2], red[3]));
        if (m) atomicMax(word, m);
    }
}

// w_t·x_t of the labelled rows as an operand with rows h and k = t, one scale for all (from the word that pack_rows
// left). One workgroup turns 32 rows x 64 columns. Rows without a label are not read, so that nothing in them counts.
__global__ __launch_bounds__(256) void pack_weighted_kernel(const float* __restrict__ x, const float* __restrict__ weights,
                                                            const int* __restrict__ row_of, const unsigned* words, int K,
                                                            _Float16* __restrict__ out, int steps) {
    constexpr int PITCH = 65;
    __shared__ unsigned turn[32 * PITCH];
    const int count = (int)words[WORD_COUNT], b = blockIdx.x, c0 = blockIdx.y * 64;
    if (32 * b >= count) return;
    const int tid = threadIdx.x, r = tid >> 3, o = tid & 7, j = 32 * b + r;
    const float sc = exp2_int(pair_scale_exp(words[WORD_WX]));
    float v[8] = {};
    if (j < count) {
        const int from = row_of[j];
        load8(x + (size_t)from * K, c0 + o * 8, K, v);
        const float w = weights ? weights[from] : 1.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        _Float16 h, l;
        split_value(v[i] * sc, h, l);
        turn[r * PITCH + o * 8 + i] =
            (unsigned)__builtin_bit_cast(unsigned short, h) | (unsigned)__builtin_bit_cast(unsigned short, l) << 16;
    }
    __syncthreads();
    const int h = tid & 63, u = tid >> 6, hg = (c0 + h) >> 5;
    if (hg >= (K + 31) / 32) return;
    f16x8 th, tl;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned w = turn[(8 * u + i) * PITCH + h];
        th[i] = __builtin_bit_cast(_Float16, (unsigned short)w);
        tl[i] = __builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
    }
    _Float16* at = out + ((size_t)hg * steps + b) * (4 * FRAG) + unit_at<2>(h & 31, u);
    *reinterpret_cast<f16x8*>(at) = th;
    *reinterpret_cast<f16x8*>(at + FRAG) = tl;
}

// ------------------------------------------------------------------------------- logits and what they become

struct Targets {
    const int *row_of, *targets;
    float* z_target;           // [labelled row]
};
struct Logits {
    Operand W, x;              // W's piece: rows v; x: rows t
    const int *ew, *ex;        // their rows' scale exponents
    const float* bias;         // padded to whole tiles, −∞ behind the piece
    const unsigned* words;
    int v0, vocab;             // the piece's first row, its rows
};

// Tiles are taken in groups of 8 vocabulary tiles, all token tiles of a group before the next: 32 tiles in a row, what
// an XCD runs at a time, share 8 of W's panels and 4 of x's.
__device__ __forceinline__ void grouped_tile(int u, int tiles_v, int tiles_t, int& tv, int& tt) {
    const int per = 8 * tiles_t, g = u / per, first = 8 * g, width = min(8, tiles_v - first), in = u - g * per;
    tt = in / width;
    tv = first + in - tt * width;
}

// The wave's logits from its accumulators, in place; `v` and `t`: the first of the wave's rows and columns.
template <int BM, int BN>
__device__ __forceinline__ void to_logits(const Logits& p, f32x4 (&acc)[BM][BN], int v, int t, int lane) {
    int ex[BN];
#pragma unroll
    for (int j = 0; j < BN; ++j) ex[j] = p.ex[t + 16 * j + (lane & 15)];
#pragma unroll
    for (int i = 0; i < BM; ++i) {
        const int at = v + 16 * i + 4 * (lane >> 4);
        const int4 ew = *reinterpret_cast<const int4*>(p.ew + at);
        const f32x4 b = *reinterpret_cast<const f32x4*>(p.bias + at);
        const int e[4] = {ew.x, ew.y, ew.z, ew.w};
#pragma unroll
        for (int j = 0; j < BN; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_amdgcn_ldexpf(acc[i][j][r], -(e[r] + ex[j])) + b[r];
    }
}

// Each tile's maximum and Σ exp(z − maximum) for every row (token): part[tile_v][t]. The target's logit, where the tile has
// it, goes to z_target[t]: the one that is in the sum, so that what its product is off by cancels in a small loss.
template <class C, int PW>
__global__ __launch_bounds__(C::THREADS, C::PER_CU) void vocab_stats_kernel(Logits p, Targets y,
                                                                                        float2* __restrict__ part, int pitch) {
    typedef typename C::template Tile<PW, 2> T;
    constexpr int SIZE = C::SIZE, BM = C::BM, BN = C::BN;
    __shared__ __attribute__((aligned(16))) _Float16 lds[T::LDS_HALVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave / C::WN, wn = wave % C::WN;
    const int count = (int)p.words[WORD_COUNT];
    const int tiles_t = (count + SIZE - 1) / SIZE, tiles_v = (p.vocab + SIZE - 1) / SIZE, units = tiles_v * tiles_t;
    p.x.groups = (count + 31) / 32;
    for (int n = 0;; ++n) {
        const int u = unit_of(n);
        if (n * (int)gridDim.x >= units) break;
        if (u >= units) continue;
        int tv, tt;
        grouped_tile(u, tiles_v, tiles_t, tv, tt);
        typename T::Acc acc;
        T::product(p.W, p.x, tv * T::MG, tt * T::NG, 0, p.W.steps, lds, acc, wave, lane);
        const int v = tv * SIZE + wm * C::WM_ROWS, t = tt * SIZE + wn * C::WN_COLS;
        to_logits(p, acc, v, t, lane);
#pragma unroll
        for (int j = 0; j < BN; ++j) {
            const int at = t + 16 * j + (lane & 15);
            const int where = (at < count ? y.targets[y.row_of[at]] : -1) - (p.v0 + v + 4 * (lane >> 4));
            if (!__any(where >= 0 && where < 16 * BM)) continue;
#pragma unroll
            for (int i = 0; i < BM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (where == 16 * i + r) y.z_target[at] = acc[i][j][r];
        }
        float2* red = reinterpret_cast<float2*>(lds);
#pragma unroll
        for (int j = 0; j < BN; ++j) {
            float m = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < BM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[i][j][r]);
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float at = m == -__builtin_inff() ? 0.0f : m;
            float s[4] = {};
#pragma unroll
            for (int i = 0; i < BM; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[r] += __builtin_amdgcn_exp2f((acc[i][j][r] - at) * LOG2E);
            float sum = (s[0] + s[1]) + (s[2] + s[3]);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (lane < 16) red[wm * SIZE + wn * C::WN_COLS + 16 * j + lane] = make_float2(m, sum);
        }
        __syncthreads();
        if (threadIdx.x < SIZE) {
            const float2 a = red[threadIdx.x], b = red[SIZE + threadIdx.x];
            const float m = fmaxf(a.x, b.x), at = m == -__builtin_inff() ? 0.0f : m;
            const float sum = a.y * __builtin_amdgcn_exp2f((a.x - at) * LOG2E) +
                              b.y * __builtin_amdgcn_exp2f((b.x - at) * LOG2E);
            part[(size_t)(p.v0 / SIZE + tv) * pitch + tt * SIZE + threadIdx.x] = make_float2(m, sum);
        }
        __syncthreads();
    }
}

// Σ w·L of the labelled rows, in an order of its own: one workgroup of N threads.
template <int N>
__device__ __forceinline__ void total_loss(const int* row_of, int count, const float* row_loss, const float* weights,
                                           float scale, float* loss) {
    __shared__ double red[N / 64];
    double s = 0.0;
    for (int k = threadIdx.x; k < count; k += N) {
        const int r = row_of[k];
        s += (double)__hip_atomic_load(row_loss + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) *
             (weights ? (double)weights[r] : 1.0);
    }
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int k = 0; k < N / 64; ++k) s += red[k];
        *loss = (float)(s * (double)scale);
    }
}
__global__ __launch_bounds__(1024) void vocab_total_kernel(const int* row_of, const unsigned* words,
                                                           const float* row_loss, const float* weights, float scale,
                                                           float* loss) {
    total_loss<1024>(row_of, (int)words[WORD_COUNT], row_loss, weights, scale, loss);
}

// One wave a labelled row: the tiles' statistics merged, less the target's logit. With `loss` the last workgroup to end sums
// the rows' weighted losses.
__global__ __launch_bounds__(256) void vocab_merge_kernel(const float2* __restrict__ part, int pitch, int tiles,
                                                          unsigned* words, const int* __restrict__ row_of,
                                                          const float* __restrict__ z_target, float* row_loss,
                                                          float* __restrict__ lse, const float* __restrict__ weights,
                                                          float scale, float* loss) {
    const int j = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63, count = (int)words[WORD_COUNT];
    if (j < count) {
        const int r = row_of[j];
        const float z = z_target[j];
        // Each lane's tiles, four at a time: the maximum and the sum so far.
        float m = -__builtin_inff(), s = 0.0f;
        for (int k = lane; k < tiles; k += 256) {
            float2 a[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                a[q] = k + 64 * q < tiles ? part[(size_t)(k + 64 * q) * pitch + j] : make_float2(-__builtin_inff(), 0.0f);
            const float top = fmaxf(fmaxf(m, fmaxf(a[0].x, a[1].x)), fmaxf(a[2].x, a[3].x));
            const float at = top == -__builtin_inff() ? 0.0f : top;
            s *= __builtin_amdgcn_exp2f((m - at) * LOG2E);
#pragma unroll
            for (int q = 0; q < 4; ++q) s = fmaf(a[q].y, __builtin_amdgcn_exp2f((a[q].x - at) * LOG2E), s);
            m = top;
        }
        float top = m;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float at = top == -__builtin_inff() ? 0.0f : top;
        const double sum = wave_sum_d((double)(s * __builtin_amdgcn_exp2f((m - at) * LOG2E)));
        if (lane == 0) {
            const double l = log(sum);
            lse[r] = (float)((double)top + l);
            __hip_atomic_store(row_loss + r, (float)(((double)top - (double)z) + l), __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (!loss) return;
    __shared__ unsigned last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(words + WORD_ENDED, 1u) + 1 == gridDim.x;
    __syncthreads();
    if (!last) return;
    __threadfence();
    total_loss<256>(row_of, count, row_loss, weights, scale, loss);
}

struct GradOut {
    const int *row_of, *targets;
    const float *lse, *weights;
    _Float16* g;     // rows t, columns v: G·2^G_SCALE
    int steps_v, groups_t;
    float* db_part;  // [4 a token tile][padded piece] (null: no bias gradient)
    int db_pitch;
};

// A piece's G, packed as it lies in the accumulators (a lane has four v of one t in a row).
template <class C, int PW, bool DB>
__global__ __launch_bounds__(C::THREADS, C::PER_CU) void vocab_grad_kernel(Logits p, GradOut g) {
    typedef typename C::template Tile<PW, 2> T;
    constexpr int SIZE = C::SIZE, BM = C::BM, BN = C::BN;
    __shared__ __attribute__((aligned(16))) _Float16 lds[T::LDS_HALVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave / C::WN, wn = wave % C::WN;
    const int count = (int)p.words[WORD_COUNT];
    const int tiles_t = (count + SIZE - 1) / SIZE, tiles_v = (p.vocab + SIZE - 1) / SIZE, units = tiles_v * tiles_t;
    p.x.groups = (count + 31) / 32;
    for (int n = 0;; ++n) {
        const int u = unit_of(n);
        if (n * (int)gridDim.x >= units) break;
        if (u >= units) continue;
        int tv, tt;
        grouped_tile(u, tiles_v, tiles_t, tv, tt);
        typename T::Acc acc;
        T::product(p.W, p.x, tv * T::MG, tt * T::NG, 0, p.W.steps, lds, acc, wave, lane);
        const int v = tv * SIZE + wm * C::WM_ROWS, t = tt * SIZE + wn * C::WN_COLS;
        to_logits(p, acc, v, t, lane);
        float w[BN];
#pragma unroll
        for (int j = 0; j < BN; ++j) {
            const int at = t + 16 * j + (lane & 15);
            const bool live = at < count;
            const int r = live ? g.row_of[at] : 0;
            const float lse = live ? g.lse[r] : 0.0f;
            if (DB) w[j] = live ? (g.weights ? g.weights[r] : 1.0f) : 0.0f;
            // The target's place among the lane's values: 16·i + e.
            const int y = (live ? g.targets[r] : -1) - (p.v0 + v + 4 * (lane >> 4));
#pragma unroll
            for (int i = 0; i < BM; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = __builtin_amdgcn_exp2f((acc[i][j][e] - lse) * LOG2E);
                    x -= y == 16 * i + e ? 1.0f : 0.0f;
                    acc[i][j][e] = live ? x * (float)(1 << G_SCALE) : 0.0f;
                }
        }
#pragma unroll
        for (int i = 0; i < BM / 2; ++i) {
            const int vg = (v >> 5) + i;
            if (vg >= g.steps_v) break;  // wave-uniform
#pragma unroll
            for (int j = 0; j < BN / 2; ++j) {
                const int tg = (t >> 5) + j;
                if (tg >= g.groups_t) break;  // wave-uniform
                f32x4 c[2][2];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int k = 0; k < 2; ++k) c[q][k] = acc[2 * i + q][2 * j + k];
                store_transposed(c, g.g + ((size_t)tg * g.steps_v + vg) * (4 * FRAG), lane);
            }
            if constexpr (DB) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    f32x4 db = {};
#pragma unroll
                    for (int j = 0; j < BN; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) db[e] = fmaf(acc[2 * i + q][j][e], w[j], db[e]);
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1)
#pragma unroll
                        for (int e = 0; e < 4; ++e) db[e] += __shfl_xor(db[e], o, 64);
                    if ((lane & 15) == 0)
                        *reinterpret_cast<f32x4*>(g.db_part + (size_t)(tt * C::WN + wn) * g.db_pitch + vg * 32 + 16 * q +
                                                  4 * (lane >> 4)) = db;
                }
            }
        }
    }
}

struct GradProducts {
    Operand g;         // rows t, columns v
    Operand wx;        // rows h, columns t: dW = gᵀ·wxᵀ over t
    Operand W;         // rows v, columns h: dx = g·W over v
    unsigned* words;
    int vocab, hidden; // the piece's rows, the width
    float* dW;         // the piece's first row
    float scale;
    float* dx_part;    // [split][padded rows][hidden]
    int cap_rows;      // Σ over the splits of padded rows that dx_part holds (0: no dx)
    int first;         // the first piece stores, the others add
    int steps_first, units_first;  // the first piece's steps over v and units of dW, which say how dx's sum is split
    int tiles_v, tiles_h;
    float* dw_part;    // [split][the piece's rows][hidden]: dW's partial sums, when its sum is split
    int most_e;        // splits that dw_part holds (1: none)
};

struct Splits {
    int x, e;
};
// The ways that dx's sum over a piece and dW's over the rows are split: those whose longest worker ends first. Worker w of
// G takes units w, w + G, …: dW's, then dx's; the longest is the first of a class of equals. A small table has few tiles
// of dW and, with many rows, long ones: 15320 x 768 x 2304 took 1.6 ms with 27 whole ones, 0.8 with them split.
// Every wave plans for itself, a pair of splits a lane at a time.
__device__ __forceinline__ Splits plan_splits(const GradProducts& p, int count, int G, int lane) {
    const int tiles_t = (count + TILE - 1) / TILE, steps_t = (count + 31) / 32, steps_v = p.steps_first;
    const int most = p.cap_rows ? max(1, min(min(MAX_SPLITS, steps_v), p.cap_rows / max(tiles_t * TILE, 1))) : 1;
    const int most_e = max(1, min(p.most_e, steps_t / 8));
    unsigned long long best = ~0ull;
    for (int k = lane; k < most * most_e; k += 64) {
        const int se = k / most + 1, s = k - (se - 1) * most + 1;
        const int ne = p.units_first * se, le = (steps_t + se - 1) / se + (se > 1 ? 4 : 0);
        const int units = ne + (p.cap_rows ? tiles_t * p.tiles_h * s : 0), lx = (steps_v + s - 1) / s;
        unsigned long long time = 0;
        for (int w = 0; w < G; w = w == 0 && ne % G != 0 ? ne % G : G) {
            const int mine = (units - w + G - 1) / G, e = max(0, (ne - w + G - 1) / G);
            // Each unit costs about 24 steps beside its own: the first copies, the stores.
            time = max(time, (unsigned long long)e * (le + 24) + (unsigned long long)(mine - e) * (lx + 24));
        }
        best = min(best, time << 16 | (unsigned)(k & 0xffff));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) best = min(best, (unsigned long long)__shfl_xor((long long)best, o, 64));
    const int k = (int)(best & 0xffff);
    return {__builtin_amdgcn_readfirstlane(k % most + 1), __builtin_amdgcn_readfirstlane(k / most + 1)};
}

// Four values of a row of which `left` more follow.
__device__ __forceinline__ f32x4 load4(const float* at, int left) {
    f32x4 v = {};
    if (left >= 4) {
        v = *reinterpret_cast<const f32x4_any*>(at);
    } else if (left > 0) {
#pragma unroll
        for (int r = 0; r < 3; ++r)
            if (r < left) v[r] = at[r];
    }
    return v;
}
__device__ __forceinline__ void store4(float* at, int left, f32x4 v) {
    if (left >= 4) {
        *reinterpret_cast<f32x4_any*>(at) = v;
    } else if (left > 0) {
#pragma unroll
        for (int r = 0; r < 3; ++r)
            if (r < left) at[r] = v[r];
    }
}

// out[row, h …] (+)= acc·2^e·scale: a lane's values are four neighbours h of the rows row + 16·j. What a row block adds to
// is read two blocks ahead of its stores.
template <int BM, int BN>
__device__ __forceinline__ void put_tile(const f32x4 (&acc)[BM][BN], float* out, int row, int rows, int h, int hidden,
                                         bool add, int e, float scale) {
    f32x4 old[3][BN];
    auto fetch = [&](int i) {
#pragma unroll
        for (int j = 0; j < BN; ++j)
            old[i % 3][j] = add && row + 16 * j < rows
                                ? load4(out + (size_t)(row + 16 * j) * hidden + h + 16 * i, hidden - h - 16 * i)
                                : f32x4{};
    };
    fetch(0);
    fetch(1);
#pragma unroll
    for (int i = 0; i < BM; ++i) {
        if (i + 2 < BM) fetch(i + 2);
#pragma unroll
        for (int j = 0; j < BN; ++j) {
            f32x4 v = old[i % 3][j];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += __builtin_amdgcn_ldexpf(acc[i][j][r], e) * scale;
            if (row + 16 * j < rows) store4(out + (size_t)(row + 16 * j) * hidden + h + 16 * i, hidden - h - 16 * i, v);
        }
    }
}

// Both products of a piece in one launch, transposed: the columns h are the accumulators' rows, four in a row of a lane,
// so that what is read and written of dW and dx goes 16 bytes at a time.
template <int PW>
__global__ __launch_bounds__(512, 1) void vocab_products_kernel(GradProducts p) {
    typedef T256 C;
    typedef typename C::template Tile<2, 2, false, true> TE;
    typedef typename C::template Tile<PW, 2, true, false> TX;
    __shared__ __attribute__((aligned(16))) _Float16 lds[TE::LDS_HALVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave / C::WN, wn = wave % C::WN;
    const int count = (int)p.words[WORD_COUNT];
    if (count == 0) return;
    const int tiles_t = (count + TILE - 1) / TILE, steps_v = p.g.steps, steps_t = (count + 31) / 32;
    const Splits plan = plan_splits(p, count, gridDim.x, lane);
    const int splits = p.cap_rows ? plan.x : 0, splits_e = plan.e;
    const int tiles_e = p.tiles_v * p.tiles_h, units_e = tiles_e * splits_e;
    const int units = units_e + tiles_t * p.tiles_h * splits;
    const int e_wx = -(G_SCALE + pair_scale_exp(p.words[WORD_WX])), e_w = -(G_SCALE + pair_scale_exp(p.words[WORD_W]));
    p.g.groups = steps_t;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.words[WORD_SPLITS] = splits;
        p.words[WORD_SPLITS_E] = splits_e;
    }
    for (int n = 0;; ++n) {
        const int u = unit_of(n);
        if (n * (int)gridDim.x >= units) break;
        if (u >= units) continue;
        typename TE::Acc acc;
        if (u < units_e) {
            const int se = u / tiles_e, in = u - se * tiles_e, tv = in / p.tiles_h, th = in - tv * p.tiles_h;
            const int s0 = (int)((long)steps_t * se / splits_e), s1 = (int)((long)steps_t * (se + 1) / splits_e);
            TE::product(p.wx, p.g, th * TE::MG, tv * TE::NG, s0, s1, lds, acc, wave, lane);
            put_tile(acc, splits_e > 1 ? p.dw_part + (size_t)se * p.vocab * p.hidden : p.dW,
                     tv * TILE + wn * C::WN_COLS + (lane & 15), p.vocab, th * TILE + wm * C::WM_ROWS + 4 * (lane >> 4),
                     p.hidden, splits_e == 1, e_wx, p.scale);
        } else {
            const int w = u - units_e, per = tiles_t * p.tiles_h, s = w / per, in = w - s * per;
            const int tt = in / p.tiles_h, th = in - tt * p.tiles_h;
            const int s0 = (int)((long)steps_v * s / splits), s1 = (int)((long)steps_v * (s + 1) / splits);
            TX::product(p.W, p.g, th * TX::MG, tt * TX::NG, s0, s1, lds, acc, wave, lane);
            put_tile(acc, p.dx_part + (size_t)s * tiles_t * TILE * p.hidden,
                     tt * TILE + wn * C::WN_COLS + (lane & 15), tiles_t * TILE,
                     th * TILE + wm * C::WM_ROWS + 4 * (lane >> 4), p.hidden, !p.first, e_w, 1.0f);
        }
    }
}

// dW += Σ over the splits of its sum, where it was split.
__global__ __launch_bounds__(256) void vocab_dw_kernel(const float* __restrict__ part, const unsigned* words, size_t n,
                                                       float* __restrict__ dW) {
    const int splits = (int)words[WORD_SPLITS_E];
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (splits < 2 || i >= n) return;
    float s = 0.0f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) s += part[k * n + i];
    dW[i] += s;
}

// dx_r = w_r·scale·Σ over the splits, 0 for rows without a label.
__global__ __launch_bounds__(256) void vocab_dx_kernel(const float* __restrict__ part, const unsigned* words,
                                                       const int* __restrict__ place,
                                                       const float* __restrict__ weights, float scale, int hidden,
                                                       float* __restrict__ dx) {
    const int r = blockIdx.x, j = place[r], count = (int)words[WORD_COUNT], splits = (int)words[WORD_SPLITS];
    const size_t stride = (size_t)((count + TILE - 1) / TILE * TILE) * hidden;
    const float f = (weights ? weights[r] : 1.0f) * scale;
    for (int h = threadIdx.x; h < hidden; h += 256) {
        float s = 0.0f;
        if (j >= 0) {
#pragma unroll 8
            for (int k = 0; k < splits; ++k) s += part[k * stride + (size_t)j * hidden + h];
            s *= f;
        }
        dx[(size_t)r * hidden + h] = s;
    }
}

__global__ __launch_bounds__(256) void vocab_db_kernel(const float* __restrict__ part, int pitch, const unsigned* words,
                                                       int vocab, float scale, float* __restrict__ db) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= vocab) return;
    const int n = ((int)words[WORD_COUNT] + 63) / 64;
    double s = 0.0;
#pragma unroll 8
    for (int k = 0; k < n; ++k) s += part[(size_t)k * pitch + v];
    db[v] += (float)(s * (double)scale * (1.0 / (1 << G_SCALE)));
}

// ------------------------------------------------------------------------------------------ launches

long pad_tile(long n) { return (n + TILE - 1) / TILE * TILE; }

template <typename T, int PLANES>
void launch_pack(laya_ctx* ctx, const PackRows& p, int blocks) {
    LAYA_LAUNCH((pack_rows_kernel<T, PLANES>), dim3(blocks), dim3(256), 0, ctx->stream, p);
    check_launch("pack_rows_kernel");
}

// A piece of the table: its rows' scales are their own, or all the one that `whole` says.
void pack_table(laya_ctx* ctx, const VocabArgs& a, int v0, int vocab, const unsigned* whole, int* exps, float* padded,
                _Float16* out) {
    PackRows p{};
    p.src = a.W16 ? (const void*)(a.W16 + (size_t)v0 * a.hidden) : (const void*)(a.W + (size_t)v0 * a.hidden);
    p.rows = vocab;
    p.K = a.hidden;
    p.whole = whole;
    p.exps = exps;
    p.out = out;
    p.bias = a.bias ? a.bias + v0 : nullptr;
    p.padded = padded;
    const int blocks = (int)(pad_tile(vocab) / 32);
    ProfileScope scope(ctx, "vocab_pack", 0.0, (a.W16 ? 2.0 : 4.0) * vocab * a.hidden * 2);
    if (a.W16)
        launch_pack<__bf16, 1>(ctx, p, blocks);
    else
        launch_pack<float, 2>(ctx, p, blocks);
}

void table_amax(laya_ctx* ctx, const VocabArgs& a, unsigned* word) {
    const size_t n = (size_t)a.vocab * a.hidden;
    ProfileScope scope(ctx, "vocab_amax", 0.0, (a.W16 ? 2.0 : 4.0) * n);
    const dim3 grid(blocks_for(n, 16384, 2048));
    if (a.W16)
        LAYA_LAUNCH(table_amax_kernel<__bf16>, grid, dim3(256), 0, ctx->stream, a.W16, n, word);
    else
        LAYA_LAUNCH(table_amax_kernel<float>, grid, dim3(256), 0, ctx->stream, a.W, n, word);
    check_launch("table_amax_kernel");
}

void pack_states(laya_ctx* ctx, const VocabArgs& a, const int* row_of, unsigned* words, int* exps, _Float16* out,
                 bool weighted) {
    PackRows p{};
    p.src = a.x;
    p.row_of = row_of;
    p.count = words + WORD_COUNT;
    p.rows = a.rows;
    p.K = a.hidden;
    p.exps = exps;
    p.out = out;
    if (weighted) {
        p.weights = a.row_weights;
        p.wx = words + WORD_WX;
    }
    launch_pack<float, 2>(ctx, p, groups_of(a.rows));
}

// Rows of the vocabulary a piece takes: whole tiles, pieces of about equal size, `each` bytes a row. Under a memory cap no
// more than fits what the cap leaves beside the `fixed` bytes of the workspace.
int piece_rows(const laya_ctx* ctx, int vocab, size_t each, size_t fixed) {
    size_t bytes = PIECE_BYTES;
    if (ctx->cap) {
        const size_t taken = ctx->in_use - ctx->scratch[VOCAB_SLOT].bytes + fixed + (64 << 10);
        bytes = std::min(bytes, ctx->cap > taken ? ctx->cap - taken : 0);
    }
    const long most = std::max<long>(TILE, (long)(bytes / each) / TILE * TILE);
    const long pieces = (vocab + most - 1) / most;
    return (int)std::min<long>(pad_tile((vocab + pieces - 1) / pieces), pad_tile(vocab));
}

template <class C>
int workgroups(const laya_ctx* ctx) { return std::max(8, ctx->cu_count / 8 * 8) * C::PER_CU; }

// f(the tile of a launch of `rows` x `vocab` logits). A round of 256 tiles over the chip takes about as long as three units a
// CU of 128 tiles (57 us and 19 us over 768 columns), which fill the last round better, two to a CU hide each other's ends,
// and a small problem gets on more CUs: 600 rows x 50368 stats 131 us on 128 and 173 on 256, 400 rows 119 and 115, 4915
// rows 976 and 925; 487 x 7905 34 and 57.
template <class F> void with_tile(laya_ctx* ctx, long rows, long vocab, F&& f) {
    const long G = workgroups<T256>(ctx), large = pad_tile(rows) / 256 * (pad_tile(vocab) / 256),
               small = (rows + 127) / 128 * ((vocab + 127) / 128);
    const double by_small = std::max(0.6, (double)small / (3.0 * G) + 0.15);
    if (by_small < (double)((large + G - 1) / G))
        f(T128());
    else
        f(T256());
}

}  // namespace

void vocab_merge(laya_ctx* ctx, const VocabArgs& a, const float2* part, int pitch, int tiles, unsigned* words,
                 const int* row_of, const float* z_target, float* row_loss, float* lse, float* loss) {
    // The total by the last workgroup saves a launch (4 of 52 µs at 19 rows), but its fences cost 0.07 µs a workgroup, one
    // after another: 250 µs at 13871 rows, where a launch of its own takes 6.
    const bool own = a.rows > VOCAB_FEW;
    LAYA_LAUNCH(vocab_merge_kernel, dim3((a.rows + 3) / 4), dim3(256), 0, ctx->stream, part, pitch, tiles, words, row_of,
                z_target, row_loss, lse, a.row_weights, a.scale, own ? nullptr : loss);
    check_launch("vocab_merge_kernel");
    if (loss && own) {
        LAYA_LAUNCH(vocab_total_kernel, dim3(1), dim3(1024), 0, ctx->stream, row_of, words, row_loss, a.row_weights,
                    a.scale, loss);
        check_launch("vocab_total_kernel");
    }
}

void vocab_ce_fwd(laya_ctx* ctx, const VocabArgs& a, float* row_loss, float* lse, float* loss, int* bad_count) {
    if (a.rows == 0) {
        if (loss) fill(ctx, loss, 0.0f, 1);
        if (bad_count) fill(ctx, reinterpret_cast<float*>(bad_count), 0.0f, 1);
        return;
    }
    if (vocab_few_rows(a)) return vocab_few_fwd(ctx, a, row_loss, lse, loss, bad_count);
    const int planes = a.W16 ? 1 : 2, pitch = (int)pad_tile(a.rows);
    const int most_tiles = (a.vocab + 127) / 128;
    const int piece = piece_rows(ctx, a.vocab, (size_t)steps_of(a.hidden) * 64 * planes + 8,
                                 2 * halves(a.rows, a.hidden, 2) + 8 * ((size_t)most_tiles + 2) * pitch);
    unsigned* words;
    int *row_of, *ex, *ew;
    float *padded, *z_target;
    _Float16 *xp, *wp;
    float2* part;
    carve(ctx, VOCAB_SLOT, [&](Carve& ws) {
        ws.take(words, WORDS);
        ws.take(row_of, a.rows);
        ws.take(ex, pitch);
        ws.take(ew, piece);
        ws.take(padded, piece);
        ws.take(z_target, a.rows);
        ws.take(xp, halves(a.rows, a.hidden, 2));
        ws.take(wp, halves(piece, a.hidden, planes));
        ws.take(part, (size_t)most_tiles * pitch);
    });
    LAYA_LAUNCH(label_rows_kernel, dim3(1), dim3(1024), 0, ctx->stream, a.targets, a.rows, a.vocab, row_of,
                (int*)nullptr, words, bad_count, row_loss, lse);
    check_launch("label_rows_kernel");
    pack_states(ctx, a, row_of, words, ex, xp, false);
    const Targets y{row_of, a.targets, z_target};
    int tiles = 0;
    for (int v0 = 0; v0 < a.vocab; v0 += piece) {
        const int n = std::min(piece, a.vocab - v0);
        pack_table(ctx, a, v0, n, nullptr, ew, padded, wp);
        Logits p{{wp, steps_of(a.hidden), groups_of(n)}, {xp, steps_of(a.hidden), 0}, ew, ex, padded, words, v0, n};
        ProfileScope scope(ctx, "vocab_stats", 2.0 * a.rows * a.hidden * n, 0.0);
        with_tile(ctx, a.rows, std::min(piece, a.vocab), [&](auto c) {
            typedef decltype(c) C;
            const dim3 grid(workgroups<C>(ctx)), block(C::THREADS);
            if (a.W16)
                LAYA_LAUNCH((vocab_stats_kernel<C, 1>), grid, block, 0, ctx->stream, p, y, part, pitch);
            else
                LAYA_LAUNCH((vocab_stats_kernel<C, 2>), grid, block, 0, ctx->stream, p, y, part, pitch);
            tiles = (a.vocab + C::SIZE - 1) / C::SIZE;
        });
        check_launch("vocab_stats_kernel");
    }
    vocab_merge(ctx, a, part, pitch, tiles, words, row_of, z_target, row_loss, lse, loss);
}

void vocab_ce_bwd(laya_ctx* ctx, const VocabArgs& a, const float* lse, float* dx, float* dW, float* db) {
    if (a.rows == 0) return;
    if (vocab_few_rows(a)) return vocab_few_bwd(ctx, a, lse, dx, dW, db);
    const int planes = a.W16 ? 1 : 2, pitch = (int)pad_tile(a.rows), steps_h = steps_of(a.hidden);
    const int steps_t = steps_of(a.rows);
    // dx's partial sums: as many rows as its splits may come to; under a memory cap a few.
    const int cap_rows = std::max(pitch, std::min((ctx->cap ? 2 : MAX_SPLITS) * pitch, 32768));
    const int tiles_t = pitch / TILE, tiles_h = (a.hidden + TILE - 1) / TILE;
    const int piece = piece_rows(ctx, a.vocab, (size_t)steps_h * 64 * planes + (size_t)steps_t * 128 + 8 + (db ? 16 * tiles_t : 0),
                                 4 * halves(a.rows, a.hidden, 2) + 16 * (size_t)pitch +
                                     (dx ? 4 * (size_t)cap_rows * a.hidden : 0));
    // dW's partial sums: a table of few tiles, whole in one piece, takes as many splits as fill the chip twice.
    const int tiles_e = dW && piece >= a.vocab ? (a.vocab + TILE - 1) / TILE * tiles_h : 0;
    const int most_e =
        tiles_e && !ctx->cap ? std::max(1, std::min({MAX_SPLITS, 2 * workgroups<T256>(ctx) / tiles_e, steps_t / 8})) : 1;
    unsigned* words;
    int *row_of, *place, *ex, *ew;
    float *padded, *part, *db_part, *dw_part;
    _Float16 *xp, *xt, *wp, *gp;
    carve(ctx, VOCAB_SLOT, [&](Carve& ws) {
        ws.take(words, WORDS);
        ws.take(row_of, a.rows);
        ws.take(place, a.rows);
        ws.take(ex, pitch);
        ws.take(ew, piece);
        ws.take(padded, piece);
        ws.take(xp, halves(a.rows, a.hidden, 2));
        ws.take(xt, halves(a.hidden, a.rows, 2));
        ws.take(wp, halves(piece, a.hidden, planes));
        ws.take(gp, halves(a.rows, piece, 2));
        ws.take(part, dx ? (size_t)cap_rows * a.hidden : 0);
        ws.take(db_part, db ? (size_t)tiles_t * 4 * piece : 0);
        ws.take(dw_part, most_e > 1 ? (size_t)most_e * a.vocab * a.hidden : 0);
    });
    if (!db) db_part = nullptr;
    LAYA_LAUNCH(label_rows_kernel, dim3(1), dim3(1024), 0, ctx->stream, a.targets, a.rows, a.vocab, row_of, place, words,
                (int*)nullptr, (float*)nullptr, (float*)nullptr);
    check_launch("label_rows_kernel");
    pack_states(ctx, a, row_of, words, ex, xp, true);
    LAYA_LAUNCH(pack_weighted_kernel, dim3(groups_of(a.rows), (a.hidden + 63) / 64), dim3(256), 0, ctx->stream, a.x,
                a.row_weights, row_of, words, a.hidden, xt, steps_t);
    check_launch("pack_weighted_kernel");
    table_amax(ctx, a, words + WORD_W);
    int steps_v = 0, units_e = 0;
    for (int v0 = 0; v0 < a.vocab; v0 += piece) {
        const int n = std::min(piece, a.vocab - v0), tiles_v = (n + TILE - 1) / TILE;
        // Every piece splits dx's sum as the first does, so that its partial sums meet the first's.
        if (v0 == 0) {
            steps_v = steps_of(n);
            units_e = dW ? tiles_v * tiles_h : 0;
        }
        pack_table(ctx, a, v0, n, words + WORD_W, ew, padded, wp);
        Logits p{{wp, steps_h, groups_of(n)}, {xp, steps_h, 0}, ew, ex, padded, words, v0, n};
        GradOut g{row_of, a.targets, lse, a.row_weights, gp, steps_of(n), steps_t, db_part, piece};
        {
            ProfileScope scope(ctx, "vocab_grad", 2.0 * a.rows * a.hidden * n, 0.0);
            with_tile(ctx, a.rows, std::min(piece, a.vocab), [&](auto c) {
                typedef decltype(c) C;
                const dim3 grid(workgroups<C>(ctx)), block(C::THREADS);
                if (a.W16 && db)
                    LAYA_LAUNCH((vocab_grad_kernel<C, 1, true>), grid, block, 0, ctx->stream, p, g);
                else if (a.W16)
                    LAYA_LAUNCH((vocab_grad_kernel<C, 1, false>), grid, block, 0, ctx->stream, p, g);
                else if (db)
                    LAYA_LAUNCH((vocab_grad_kernel<C, 2, true>), grid, block, 0, ctx->stream, p, g);
                else
                    LAYA_LAUNCH((vocab_grad_kernel<C, 2, false>), grid, block, 0, ctx->stream, p, g);
            });
            check_launch("vocab_grad_kernel");
        }
        GradProducts q{};
        q.wx = {xt, steps_t, groups_of(a.hidden)};
        q.g = {gp, steps_of(n), 0};
        q.W = {wp, steps_h, groups_of(n)};
        q.words = words;
        q.vocab = n;
        q.hidden = a.hidden;
        q.dW = dW ? dW + (size_t)v0 * a.hidden : nullptr;
        q.scale = a.scale;
        q.dx_part = part;
        q.cap_rows = dx ? cap_rows : 0;
        q.first = v0 == 0;
        q.steps_first = steps_v;
        q.units_first = units_e;
        q.tiles_v = dW ? tiles_v : 0;
        q.tiles_h = tiles_h;
        q.dw_part = dw_part;
        q.most_e = most_e;
        if (dx || dW) {
            ProfileScope scope(ctx, "vocab_products", ((dx ? 2.0 : 0.0) + (dW ? 2.0 : 0.0)) * a.rows * a.hidden * n, 0.0);
            const dim3 grid(workgroups<T256>(ctx)), block(512);
            if (a.W16)
                LAYA_LAUNCH(vocab_products_kernel<1>, grid, block, 0, ctx->stream, q);
            else
                LAYA_LAUNCH(vocab_products_kernel<2>, grid, block, 0, ctx->stream, q);
            check_launch("vocab_products_kernel");
        }
        if (most_e > 1) {
            const size_t n_e = (size_t)a.vocab * a.hidden;
            LAYA_LAUNCH(vocab_dw_kernel, dim3((unsigned)((n_e + 255) / 256)), dim3(256), 0, ctx->stream, dw_part, words,
                        n_e, dW);
            check_launch("vocab_dw_kernel");
        }
        if (db) {
            LAYA_LAUNCH(vocab_db_kernel, dim3((n + 255) / 256), dim3(256), 0, ctx->stream, db_part, piece, words, n,
                        a.scale, db + v0);
            check_launch("vocab_db_kernel");
        }
    }
    if (dx) {
        LAYA_LAUNCH(vocab_dx_kernel, dim3(a.rows), dim3(256), 0, ctx->stream, part, words, place, a.row_weights, a.scale, a.hidden, dx);
        check_launch("vocab_dx_kernel");
    }
}

}  // namespace laya
