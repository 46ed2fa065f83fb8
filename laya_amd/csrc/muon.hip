// Newton-Schulz orthogonalisation of matrices, and the Muon step that moves parameters by it.
//
// A matrix U is brought to Frobenius norm 1 and taken through
//   A = X·Xᵀ,  X ← (a·I + b·A + c·A²)·X,   a = 3.4445, b = −4.7750, c = 2.0315
// (X with its short side n as rows, its long side m as columns): the odd quintic whose iterates push every singular
// value into about [0.7, 1.2], the coefficients of the published Muon optimizer (K. Jordan et al., 2024). All matrices
// of a call go through each of an iteration's three products in one launch:
//   gram    A  = X·Xᵀ            n x n over m, the tiles on and below the diagonal, written to both sides
//   poly    B  = a·I + b·A + c·A·A   n x n over n, likewise
//   update  X' = B·X             m x n over n, as Xᵀ·B, whose accumulators hold four columns of an X' row in a row
// X, A and B live as packed pieces alone (packed.hpp; X is read over its columns by gram and over its rows by update),
// 22 bits of every element; a·X rides on B's diagonal, so that no fp32 X is kept. Every operand is bounded (singular
// values of X at most 1.21, of A 1.46, of B 3.45), so its scale is a constant power of two and nothing is measured.
//
// Many matrices are bound by the matrix cores (three fp16 products of a fp32 one; 487 TFLOP/s of these is what a large
// library product reaches): 88 matrices of 22 layers of width 768, 110 M elements, take 5.3 ms, of which update 2.5 ms (340
// TFLOP/s; the last, 0.65 ms, also moves the parameters), gram 1.4 and poly 0.9 (270 counting one triangle, of which whole
// tiles are computed), the momentum and the norms 0.24 ms (1.3 GB at 5.5 TB/s) and packing 0.27 ms. One matrix is bound by latency: fifteen products one after another, each about
// 6 us of its K steps and 4 us of starting and ending (768 x 768: 10 us a product at any tile that fills more CUs).
#include "elementwise.hpp"
#include "packed.hpp"

namespace laya {
namespace {

using namespace packed;

constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr int SCALE = 13;  // of X, A and B: 3.45·2^13 is below fp16's largest, and 2^-37 its last bit
constexpr int NORM_CHUNK = 16384;
constexpr size_t BATCH_BYTES = (size_t)4 << 30;  // of packed matrices that a batch may take

// A run of equal matrices of a batch.
struct Shape {
    int rows, cols, count;
    int first;                // of the call's matrices (where `offsets` and `multipliers` are read)
    int n, m;                 // the short side and the long one
    int groups_n, steps_n, steps_m;
    size_t x, ab;             // a matrix's halves of X, and of A or B
    size_t x0, ab0;           // where the run's first lie
    int chunks, chunk0;       // partial sums of squares a matrix has, and where the run's first lie
    int unit0;                // the launch's units before the run
    int tiles, across;        // of a matrix, and of those a row of its tiles has (update)
    int turn;                 // the XCD that the run's first matrix goes to
};
constexpr int MAX_SHAPES = 16;

struct Batch {
    int shapes, units;
    int together;  // see find_tile
    Shape s[MAX_SHAPES];
};

struct Matrix {
    int shape, index, unit;  // the unit of its matrix
};
// The matrix that unit u belongs to, where a matrix of a shape has per(shape) units.
template <class F>
__device__ __forceinline__ Matrix find(const Batch& b, int u, F per) {
    int k = 0;
    while (k + 1 < b.shapes && u >= b.s[k + 1].unit0) ++k;
    const int in = u - b.s[k].unit0, each = per(b.s[k]);
    return {k, in / each, in % each};
}

// What a matrix's elements are before the iteration: an array's, or a Muon step's g, m (new) as u.
struct Source {
    const float* x;        // orthogonalize: the matrices one after another (null: a Muon step)
    float *grads, *momentum;
    const size_t* offsets;
    const float* coef;
    float mu;
    int nesterov, zero_grads;
};

__device__ __forceinline__ size_t base_of(const Source& f, const Shape& s, int index) {
    return f.x ? (size_t)(s.first + index) * s.rows * s.cols : f.offsets[s.first + index];
}

__device__ __forceinline__ int chunks_of(const Shape& s) { return s.chunks; }

// Σ u² of a chunk of a matrix, in double; a Muon step's momentum moves here.
__global__ __launch_bounds__(256) void muon_norm_kernel(Batch b, Source f, double* __restrict__ partial) {
    __shared__ double red[4];
    const Matrix at = find(b, blockIdx.x, chunks_of);
    const Shape& s = b.s[at.shape];
    const size_t base = base_of(f, s, at.index);
    const int size = s.rows * s.cols, lo = at.unit * NORM_CHUNK, hi = min(size, lo + NORM_CHUNK);
    const float cf = f.coef ? *f.coef : 1.0f;
    double sum = 0.0;
    if (f.x) {
        const float* x = f.x + base;
        if (((uintptr_t)x & 15u) == 0) {
            int i = lo + 4 * (int)threadIdx.x;
#pragma unroll 4
            for (; i + 3 < hi; i += 1024) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(x + i);
                sum += ((double)v[0] * v[0] + (double)v[1] * v[1]) + ((double)v[2] * v[2] + (double)v[3] * v[3]);
            }
            for (; i < hi; ++i) sum += (double)x[i] * x[i];
        } else {
            for (int i = lo + threadIdx.x; i < hi; i += 256) sum += (double)x[i] * x[i];
        }
    } else {
        const float* g = f.grads + base;
        float* m = f.momentum + base;
        auto move = [&](float gi, float mi, float& out) {
            const float gs = gi * cf;
            out = fmaf(f.mu, mi, gs);
            return f.nesterov ? fmaf(f.mu, out, gs) : out;
        };
        if ((((uintptr_t)g | (uintptr_t)m) & 15u) == 0) {
            int i = lo + 4 * (int)threadIdx.x;
#pragma unroll 4
            for (; i + 3 < hi; i += 1024) {
                const f32x4 gv = *reinterpret_cast<const f32x4*>(g + i), mv = *reinterpret_cast<const f32x4*>(m + i);
                f32x4 o;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float mo;
                    const double u = move(gv[k], mv[k], mo);
                    o[k] = mo;
                    sum += u * u;
                }
                *reinterpret_cast<f32x4*>(m + i) = o;
            }
            for (; i < hi; ++i) {
                float mo;
                const double u = move(g[i], m[i], mo);
                m[i] = mo;
                sum += u * u;
            }
        } else {
            for (int i = lo + threadIdx.x; i < hi; i += 256) {
                float mo;
                const double u = move(g[i], m[i], mo);
                m[i] = mo;
                sum += u * u;
            }
        }
    }
    sum = wave_sum_d(sum);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// 32 rows x 64 columns of a matrix a block.
__device__ __forceinline__ int blocks_of(const Shape& s) { return ((s.rows + 31) / 32) * ((s.cols + 63) / 64); }

// X = U / |U|_F, packed with the short side as rows (a tall matrix is turned in LDS); a zero matrix stays zero.
__global__ __launch_bounds__(256) void muon_pack_kernel(Batch b, Source f, const double* __restrict__ partial,
                                                        _Float16* __restrict__ X) {
    constexpr int PITCH = 65;
    __shared__ unsigned turn[32 * PITCH];
    const Matrix at = find(b, blockIdx.x, blocks_of);
    const Shape& s = b.s[at.shape];
    const size_t base = base_of(f, s, at.index);
    const int across = (s.cols + 63) / 64, r0 = at.unit / across * 32, c0 = at.unit % across * 64;
    const int tid = threadIdx.x, r = tid >> 3, o = tid & 7, row = r0 + r, c = c0 + 8 * o;
    double sum = 0.0;
    const double* part = partial + s.chunk0 + (size_t)at.index * s.chunks;
    for (int k = tid & 63; k < s.chunks; k += 64) sum += part[k];
    sum = wave_sum_d(sum);
    const double inverse = sum > 0.0 ? 1.0 / sqrt(sum) : sum != sum ? sum : 0.0;
    const float cf = f.coef ? *f.coef : 1.0f;
    float v[8] = {};
    const size_t from = base + (size_t)row * s.cols;
    const float* one = f.x ? f.x : f.grads;
    const uintptr_t low = (uintptr_t)(one + from) | (f.x ? 0 : (uintptr_t)(f.momentum + from));
    if (row < s.rows && c + 8 <= s.cols && (low & 15u) == 0 && s.cols % 4 == 0) {
        f32x4 a[2], m[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) a[q] = *reinterpret_cast<const f32x4*>(one + from + c + 4 * q);
        if (!f.x) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                m[q] = *reinterpret_cast<const f32x4*>(f.momentum + from + c + 4 * q);
                if (f.zero_grads) *reinterpret_cast<f32x4*>(f.grads + from + c + 4 * q) = f32x4{};
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = a[i >> 2][i & 3];
            v[i] = f.x ? x : f.nesterov ? fmaf(f.mu, m[i >> 2][i & 3], x * cf) : m[i >> 2][i & 3];
        }
    } else if (row < s.rows) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < s.cols) {
                if (f.x) {
                    v[i] = f.x[from + c + i];
                } else {
                    const float gi = f.grads[from + c + i], m = f.momentum[from + c + i];
                    v[i] = f.nesterov ? fmaf(f.mu, m, gi * cf) : m;
                    if (f.zero_grads) f.grads[from + c + i] = 0.0f;
                }
            }
    }
    f16x8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        _Float16 h, l;
        split_value((float)((double)v[i] * inverse) * (float)(1 << SCALE), h, l);
        hi[i] = h;
        lo[i] = l;
    }
    _Float16* x = X + s.x0 + at.index * s.x;
    if (s.rows <= s.cols) {
        const int step = c >> 5;
        if (step < s.steps_m) {
            _Float16* to = x + ((size_t)(r0 >> 5) * s.steps_m + step) * (4 * FRAG) + unit_at<2>(r, o & 3);
            *reinterpret_cast<f16x8*>(to) = hi;
            *reinterpret_cast<f16x8*>(to + FRAG) = lo;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        turn[r * PITCH + o * 8 + i] = (unsigned)__builtin_bit_cast(unsigned short, (_Float16)hi[i]) |
                                      (unsigned)__builtin_bit_cast(unsigned short, (_Float16)lo[i]) << 16;
    __syncthreads();
    const int h = tid & 63, u = tid >> 6, group = (c0 + h) >> 5;
    if (group >= s.groups_n) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned w = turn[(8 * u + i) * PITCH + h];
        hi[i] = __builtin_bit_cast(_Float16, (unsigned short)w);
        lo[i] = __builtin_bit_cast(_Float16, (unsigned short)(w >> 16));
    }
    _Float16* to = x + ((size_t)group * s.steps_m + (r0 >> 5)) * (4 * FRAG) + unit_at<2>(h & 31, u);
    *reinterpret_cast<f16x8*>(to) = hi;
    *reinterpret_cast<f16x8*>(to + FRAG) = lo;
}

// ------------------------------------------------------------------------------------------ products

// Square tiles, how many workgroups share a CU, and the waves of one.
template <int SIZE_, int WAVES_N, int PER_CU_, int RING>
struct Config {
    static constexpr int SIZE = SIZE_, PER_CU = PER_CU_, WN = WAVES_N, BM = SIZE / 32, BN = SIZE / 16 / WAVES_N;
    template <bool TA> using Tile = packed::Tile<2, WAVES_N, BM, BN, 2, 2, TA, false, RING>;
};
typedef Config<256, 4, 1, 2> T256;
typedef Config<128, 2, 2, 2> T128;
typedef Config<64, 2, 2, 4> T64;

// The workgroup's tile. Of many matrices each one's tiles run on one XCD (workgroups go round the 8), so that its packed
// rows come into one L2 (22 layers: gram and poly 478 us an iteration against 578 spread); of few, a matrix's tiles go to
// the XCDs in runs (a layer's four matrices: 109 us an iteration against 118).
struct Where {
    int shape, index, tile;
};
__device__ __forceinline__ bool find_tile(const Batch& b, int u, Where& at) {
    int k = 0;
    while (k + 1 < b.shapes && u >= b.s[k + 1].unit0) ++k;
    const Shape& s = b.s[k];
    const int in = u - s.unit0;
    at.shape = k;
    if (b.together) {
        const int slot = in >> 3;
        at.index = slot / s.tiles * 8 + ((in + b.s[k].turn) & 7);
        at.tile = slot % s.tiles;
    } else {
        const int all = s.count * s.tiles, per = (all + 7) >> 3, t = (in & 7) * per + (in >> 3);
        if ((in >> 3) >= per || t >= all) return false;
        at.index = t / s.tiles;
        at.tile = t % s.tiles;
    }
    return at.index < s.count;
}

// Row ti and column tj ≤ ti of the u-th tile on or below the diagonal.
__device__ __forceinline__ void triangle_tile(int u, int& ti, int& tj) {
    ti = 0;
    while (u > ti) u -= ++ti;
    tj = u;
}

// gram (POLY false): A = X·Xᵀ; poly: B = a·I + b·A + c·A·A.
template <class C, bool POLY>
__global__ __launch_bounds__(C::template Tile<false>::THREADS, C::PER_CU) void muon_square_kernel(
    Batch b, const _Float16* __restrict__ in, _Float16* __restrict__ out) {
    typedef typename C::template Tile<false> T;
    __shared__ __attribute__((aligned(16))) _Float16 lds[T::LDS_HALVES];
    constexpr int WN = C::WN, BM = C::BM, BN = C::BN;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave / WN, wn = wave % WN;
    Where at;
    if (!find_tile(b, blockIdx.x, at)) return;
    const Shape& s = b.s[at.shape];
    int ti, tj;
    triangle_tile(at.tile, ti, tj);
    const int steps = POLY ? s.steps_n : s.steps_m;
    const _Float16* from = in + (POLY ? s.ab0 + at.index * s.ab : s.x0 + at.index * s.x);
    _Float16* to = out + s.ab0 + at.index * s.ab;
    const Operand op{from, steps, s.groups_n};
    typename T::Acc acc;
    T::product(op, op, ti * T::MG, tj * T::NG, 0, steps, lds, acc, wave, lane);
    unsigned* turn = reinterpret_cast<unsigned*>(lds) + wave * TURN_DWORDS;
    const int i0 = ti * C::SIZE + wm * BM * 16, j0 = tj * C::SIZE + wn * BN * 16;
#pragma unroll
    for (int i = 0; i < BM / 2; ++i)
#pragma unroll
        for (int j = 0; j < BN / 2; ++j) {
            const int gi = (i0 >> 5) + i, gj = (j0 >> 5) + j;
            if (gi >= s.groups_n || gj >= s.groups_n) continue;  // wave-uniform
            const size_t below = ((size_t)gi * s.steps_n + gj) * (4 * FRAG), above = ((size_t)gj * s.steps_n + gi) * (4 * FRAG);
            f32x4 c[2][2];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    c[q][k] = acc[2 * i + q][2 * j + k] * (POLY ? NS_C / (1 << SCALE) : 1.0f / (1 << SCALE));
                    if constexpr (POLY) {
                        const _Float16* a = from + above + unit_at<2>(16 * k + (lane & 15), 2 * q + (lane >> 5)) +
                                            4 * ((lane >> 4) & 1);
                        const f32x4 hi = __builtin_convertvector(*reinterpret_cast<const f16x4*>(a), f32x4);
                        const f32x4 lo = __builtin_convertvector(*reinterpret_cast<const f16x4*>(a + FRAG), f32x4);
                        const int col = 32 * gj + 16 * k + (lane & 15) - (32 * gi + 16 * q + 4 * (lane >> 4));
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            c[q][k][e] = fmaf(NS_B, hi[e] + lo[e], c[q][k][e]) + (col == e ? NS_A * (1 << SCALE) : 0.0f);
                    }
                }
            store_transposed(c, to + above, lane);
            if (ti != tj) {
                turn_write(c, turn, lane);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    f16x8 hi, lo;
                    turn_read(turn, lane, q, hi, lo);
                    _Float16* p = to + below + unit_at<2>(16 * q + (lane & 15), lane >> 4);
                    *reinterpret_cast<f16x8*>(p) = hi;
                    *reinterpret_cast<f16x8*>(p + FRAG) = lo;
                }
            }
        }
}

// What the last update writes: the matrices, or parameters moved by them.
struct Sink {
    float* out;              // orthogonalize (null: a Muon step)
    float* params;
    const size_t* offsets;
    const float* multipliers;
    float rate, decay;       // p = decay·p − rate·multiplier·X
};

// X' = B·X; LAST: into the sink.
template <class C, bool LAST>
__global__ __launch_bounds__(C::template Tile<true>::THREADS, C::PER_CU) void muon_update_kernel(
    Batch b, const _Float16* __restrict__ X, const _Float16* __restrict__ B, _Float16* __restrict__ out, Sink sink) {
    typedef typename C::template Tile<true> T;
    __shared__ __attribute__((aligned(16))) _Float16 lds[T::LDS_HALVES];
    constexpr int WN = C::WN, BM = C::BM, BN = C::BN;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave / WN, wn = wave % WN;
    Where at;
    if (!find_tile(b, blockIdx.x, at)) return;
    const Shape& s = b.s[at.shape];
    // Tiles in strips of 6 columns, row by row, so that a run of them shares rows and columns.
    const int down = s.tiles / s.across, strip = at.tile / (6 * down), wide = min(6, s.across - 6 * strip);
    const int in_strip = at.tile - strip * 6 * down, ti = in_strip / wide, tj = 6 * strip + in_strip % wide;
    const Operand x{X + s.x0 + at.index * s.x, s.steps_m, s.groups_n}, bb{B + s.ab0 + at.index * s.ab, s.steps_n, s.groups_n};
    typename T::Acc acc;
    T::product(x, bb, ti * T::MG, tj * T::NG, 0, s.steps_n, lds, acc, wave, lane);
    const int i0 = ti * C::SIZE + wm * BM * 16, j0 = tj * C::SIZE + wn * BN * 16;  // i over m, j over n
    if constexpr (!LAST) {
        _Float16* to = out + s.x0 + at.index * s.x;
#pragma unroll
        for (int i = 0; i < BM / 2; ++i)
#pragma unroll
            for (int j = 0; j < BN / 2; ++j) {
                const int gi = (i0 >> 5) + i, gj = (j0 >> 5) + j;
                if (gi >= s.steps_m || gj >= s.groups_n) continue;  // wave-uniform
                f32x4 c[2][2];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int k = 0; k < 2; ++k) c[q][k] = acc[2 * i + q][2 * j + k] * (1.0f / (1 << SCALE));
                store_transposed(c, to + ((size_t)gj * s.steps_m + gi) * (4 * FRAG), lane);
            }
    } else {
        constexpr float unscale = 1.0f / ((float)(1 << SCALE) * (float)(1 << SCALE));
        const int which = s.first + at.index;
        const size_t base = sink.out ? (size_t)which * s.rows * s.cols : sink.offsets[which];
        float* to = (sink.out ? sink.out : sink.params) + base;
        const float k = sink.out ? unscale : -sink.rate * sink.multipliers[which] * unscale;
        const bool wide = s.rows <= s.cols, vec = wide && s.cols % 4 == 0 && ((uintptr_t)to & 15u) == 0;
        // A row block's old values are read together, so that their latencies overlap.
#pragma unroll
        for (int i = 0; i < BM; ++i) {
            const int col = i0 + 16 * i + 4 * (lane >> 4), row = j0 + (lane & 15);  // of X; block j: row + 16·j
            f32x4 old[BN];
            if (!sink.out) {
#pragma unroll
                for (int j = 0; j < BN; ++j) {
                    const int r = min(row + 16 * j, s.n - 1);
                    if (vec) {
                        old[j] = *reinterpret_cast<const f32x4*>(to + (size_t)r * s.cols + min(col, s.m - 4));
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int c = min(col + e, s.m - 1);
                            old[j][e] = to[wide ? (size_t)r * s.cols + c : (size_t)c * s.cols + r];
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < BN; ++j) {
                const int r = row + 16 * j;
                f32x4 v = acc[i][j] * k;
                if (!sink.out) v += old[j] * sink.decay;
                if (r >= s.n) continue;
                if (vec) {
                    if (col < s.m) *reinterpret_cast<f32x4*>(to + (size_t)r * s.cols + col) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col + e < s.m) to[wide ? (size_t)r * s.cols + col + e : (size_t)(col + e) * s.cols + r] = v[e];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------ launches

int ceil_div(long a, long b) { return (int)((a + b - 1) / b); }

// Sets the units of a launch with tiles of size x size.
void tile_units(Batch& b, int size, bool triangle) {
    int units = 0, before = 0, matrices = 0;
    for (int k = 0; k < b.shapes; ++k) matrices += b.s[k].count;
    b.together = matrices >= 32;
    for (int k = 0; k < b.shapes; ++k) {
        Shape& s = b.s[k];
        s.across = ceil_div(s.n, size);
        s.tiles = triangle ? s.across * (s.across + 1) / 2 : ceil_div(s.m, size) * s.across;
        s.unit0 = units;
        s.turn = before & 7;
        units += b.together ? (s.count + 7) / 8 * 8 * s.tiles : (s.count * s.tiles + 7) / 8 * 8;
        before += s.count;
    }
    b.units = units;
}

// The tile for a launch, by an estimate of its time. A tile of K / 32 steps takes about alone·(steps + overhead) on a CU that
// it has for itself; a full chip (whose clock the matrix cores' power then sets) gets through one in loaded·(steps +
// overhead) a CU. Microseconds on 768 x 768 to 2304 x 768 matrices, one and 88 at a time: a 256 tile 47.7 us alone over
// 24 steps and 122 over 72, a 128 tile 19.0 and 48.2, a 64 tile 10.2 and 29.2. One matrix runs its products best on 64
// tiles (10 us against 19 and 48), 22 layers gram and poly on 128 (305 + 176 us against 328 + 203 on 256) and update on
// 256 (489 against 523 on 128).
int pick_tile(laya_ctx* ctx, Batch& b, bool triangle, bool gram) {
    const struct { int size, overhead; double alone, loaded; } t[3] = {{256, 7, 1.54, 2.25}, {128, 7, 0.61, 0.7}, {64, 2, 0.40, 0.27}};
    int best = 0;
    double time = 1e30;
    for (int k = 0; k < 3; ++k) {
        tile_units(b, t[k].size, triangle);
        double total = 0, longest = 0;
        for (int q = 0; q < b.shapes; ++q) {
            const Shape& s = b.s[q];
            const double each = (gram ? s.steps_m : s.steps_n) + t[k].overhead;
            total += (double)s.count * s.tiles * each;
            longest = std::max(longest, each);
        }
        const double load = total / ctx->cu_count * t[k].loaded, one = longest * t[k].alone;
        const double cost = load > one ? load + 0.5 * one : one;  // units end unevenly: half a unit beyond the mean
        if (cost < time) {
            time = cost;
            best = k;
        }
    }
    tile_units(b, t[best].size, triangle);
    return best;
}

template <class F> void with_tile(laya_ctx* ctx, Batch& b, bool triangle, bool gram, F&& f) {
    switch (pick_tile(ctx, b, triangle, gram)) {
        case 0: return f(T256());
        case 1: return f(T128());
        default: return f(T64());
    }
}

template <bool POLY>
void launch_square(laya_ctx* ctx, Batch& b, const _Float16* in, _Float16* out) {
    double flops = 0;
    for (int k = 0; k < b.shapes; ++k)
        flops += (double)b.s[k].count * b.s[k].n * b.s[k].n * (POLY ? b.s[k].n : b.s[k].m);
    ProfileScope scope(ctx, POLY ? "muon_poly" : "muon_gram", flops, 0.0);
    with_tile(ctx, b, true, !POLY, [&](auto c) {
        typedef decltype(c) C;
        LAYA_LAUNCH((muon_square_kernel<C, POLY>), dim3(b.units), dim3(C::template Tile<false>::THREADS), 0, ctx->stream, b,
                    in, out);
    });
    check_launch("muon_square_kernel");
}

template <bool LAST>
void launch_update(laya_ctx* ctx, Batch& b, const _Float16* X, const _Float16* B, _Float16* out, const Sink& sink) {
    double flops = 0;
    for (int k = 0; k < b.shapes; ++k) flops += 2.0 * b.s[k].count * b.s[k].n * b.s[k].n * b.s[k].m;
    ProfileScope scope(ctx, "muon_update", flops, 0.0);
    with_tile(ctx, b, false, false, [&](auto c) {
        typedef decltype(c) C;
        LAYA_LAUNCH((muon_update_kernel<C, LAST>), dim3(b.units), dim3(C::template Tile<true>::THREADS), 0, ctx->stream, b, X,
                    B, out, sink);
    });
    check_launch("muon_update_kernel");
}

void run_batch(laya_ctx* ctx, Batch& b, const Source& from, const Sink& sink, int steps) {
    size_t x = 0, ab = 0;
    int chunks = 0;
    for (int k = 0; k < b.shapes; ++k) {
        Shape& s = b.s[k];
        s.n = std::min(s.rows, s.cols);
        s.m = std::max(s.rows, s.cols);
        s.groups_n = groups_of(s.n);
        s.steps_n = steps_of(s.n);
        s.steps_m = steps_of(s.m);
        s.x = halves(s.n, s.m, 2);
        s.ab = halves(s.n, s.n, 2);
        s.x0 = x;
        s.ab0 = ab;
        s.chunks = ceil_div((long)s.rows * s.cols, NORM_CHUNK);
        s.chunk0 = chunks;
        x += s.x * s.count;
        ab += s.ab * s.count;
        chunks += s.chunks * s.count;
    }
    double* partial;
    _Float16 *X[2], *A, *B;
    carve(ctx, MUON_SLOT, [&](Carve& ws) {
        ws.take(partial, chunks);
        ws.take(X[0], x);
        ws.take(X[1], x);
        ws.take(A, ab);
        ws.take(B, ab);
    });
    double elements = 0;
    for (int k = 0; k < b.shapes; ++k) elements += (double)b.s[k].count * b.s[k].rows * b.s[k].cols;
    for (int k = 0, u = 0; k < b.shapes; ++k) {
        b.s[k].unit0 = u;
        u += b.s[k].count * b.s[k].chunks;
    }
    {
        ProfileScope scope(ctx, "muon_norm", 0.0, (from.x ? 4.0 : 12.0) * elements);
        LAYA_LAUNCH(muon_norm_kernel, dim3(chunks), dim3(256), 0, ctx->stream, b, from, partial);
        check_launch("muon_norm_kernel");
    }
    int blocks = 0;
    for (int k = 0; k < b.shapes; ++k) {
        b.s[k].unit0 = blocks;
        blocks += b.s[k].count * ceil_div(b.s[k].rows, 32) * ceil_div(b.s[k].cols, 64);
    }
    {
        ProfileScope scope(ctx, "muon_pack", 0.0, (from.x ? 8.0 : 12.0) * elements);
        LAYA_LAUNCH(muon_pack_kernel, dim3(blocks), dim3(256), 0, ctx->stream, b, from, partial, X[0]);
        check_launch("muon_pack_kernel");
    }
    for (int i = 0; i < steps; ++i) {
        launch_square<false>(ctx, b, X[i & 1], A);
        launch_square<true>(ctx, b, A, B);
        if (i + 1 < steps)
            launch_update<false>(ctx, b, X[i & 1], B, X[(i + 1) & 1], sink);
        else
            launch_update<true>(ctx, b, X[i & 1], B, nullptr, sink);
    }
}

// Runs of equal matrices, taken into batches that fit the packed bytes and the shapes that a launch may name.
void run(laya_ctx* ctx, std::vector<Shape> runs, const Source& from, const Sink& sink, int steps) {
    Batch b{};
    size_t bytes = 0;
    auto flush = [&] {
        if (b.shapes) run_batch(ctx, b, from, sink, steps);
        b = Batch{};
        bytes = 0;
    };
    for (Shape s : runs) {
        const int n = std::min(s.rows, s.cols), m = std::max(s.rows, s.cols);
        const size_t each = 4 * (halves(n, m, 2) + halves(n, n, 2));
        while (s.count > 0) {
            long fit = bytes < BATCH_BYTES ? (long)((BATCH_BYTES - bytes) / each) : 0;
            if (fit == 0 && b.shapes == 0) fit = 1;
            if (fit == 0 || b.shapes == MAX_SHAPES) {
                flush();
                continue;
            }
            Shape part = s;
            part.count = (int)std::min<long>(s.count, fit);
            b.s[b.shapes++] = part;
            bytes += part.count * each;
            s.first += part.count;
            s.count -= part.count;
        }
    }
    flush();
}

}  // namespace

void orthogonalize(laya_ctx* ctx, const float* x, int count, int rows, int cols, int steps, float* out) {
    Shape s{};
    s.rows = rows;
    s.cols = cols;
    s.count = count;
    Source from{};
    from.x = x;
    Sink sink{};
    sink.out = out;
    run(ctx, {s}, from, sink, steps);
}

void muon_step(laya_ctx* ctx, const laya_matrices& mats, float* params, float* grads, float* momentum, float rate,
               float mu, int nesterov, float decay, int steps, const float* coef, int zero_grads) {
    std::vector<Shape> runs;
    for (const auto& r : mats.runs) {
        Shape s{};
        s.rows = r.rows;
        s.cols = r.cols;
        s.count = r.count;
        s.first = r.first;
        runs.push_back(s);
    }
    const Source from{nullptr, grads, momentum, mats.d_offsets, coef, mu, nesterov, zero_grads};
    const Sink sink{nullptr, params, mats.d_offsets, mats.d_multipliers, rate, decay};
    run(ctx, runs, from, sink, steps);
}

}  // namespace laya
