// Products of packed operands: the matrix-core loop of the vocabulary cross entropy (vocab.hip) and the Newton-Schulz
// iteration (muon.hip).
//
// An fp32 operand that several tiles read is split once into the fp16 pieces of split2h_4 (a power-of-two scale, then
// hi + lo, 22 bits) and kept in the order in which the matrix cores take it, so that the product's loop converts
// nothing and computes no addresses: it copies runs of memory to LDS (16 bytes a lane, no registers between) and reads
// fragments back, both linear. v_mfma_f32_32x32x16_f16 takes from lane l the 8 k of half l / 32 of row l mod 32, so a
// fragment is 32 rows x 16 k = 1 KB, [half][row][8 k], and an operand of R rows and K columns is
//   [⌈R / 32⌉ row blocks][k steps][planes: hi, lo][512 fp16]
// with zeros behind R and K, the number of k steps even (the loop takes two to a stage). bf16-valued operands keep one
// plane (split1h_4). Three piece products make one fp32-accurate product (lo·hi, hi·lo, hi·hi), two when one side has
// one plane.
#pragma once
#include "common.hpp"
#include "split.hpp"

typedef float f32x16 __attribute__((ext_vector_type(16)));

namespace laya {
namespace packed {

constexpr int FRAG = 512;  // fp16 values of a fragment

inline int row_blocks(long rows) { return (int)((rows + 31) / 32); }
inline int k_steps(long k) { return (int)((k + 31) / 32) * 2; }  // 16-deep, even
inline size_t halves(long rows, long k, int planes) { return (size_t)row_blocks(rows) * k_steps(k) * planes * FRAG; }

// A packed operand as a kernel takes it. `blocks`: its row blocks (a tile's blocks behind the last read the last).
struct Operand {
    const _Float16* data;
    int steps, blocks;
};

__device__ __forceinline__ void split_value(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// 16 bytes a lane from global memory to LDS, the wave's 64 lanes in a row from `to` (the same in every lane).
template <int OFFSET>
__device__ __forceinline__ void copy_to_lds(const _Float16* from, _Float16* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, OFFSET, 0);
}

// A workgroup of WAVES_M x WAVES_N waves, each BM x BN blocks of 32 x 32 outputs: C[m, n] += Σ_k A[m, k]·B[n, k].
template <int WAVES_M, int WAVES_N, int BM, int BN, int PA, int PB>
struct Tile {
    static constexpr int WAVES = WAVES_M * WAVES_N, THREADS = 64 * WAVES;
    static constexpr int MB = WAVES_M * BM, NB = WAVES_N * BN;  // row blocks of A and B in a tile
    static constexpr int M = 32 * MB, N = 32 * NB;
    static constexpr int A_HALVES = MB * 2 * PA * FRAG, STAGE = A_HALVES + NB * 2 * PB * FRAG;
    static constexpr int LDS_HALVES = 2 * STAGE;
    static_assert((MB + NB) % WAVES == 0, "every wave copies the same number of blocks");
    static constexpr int COPIES = (MB + NB) / WAVES;

    typedef f32x16 Acc[BM][BN];

    // Stage st (two 16-deep steps) into LDS: block b of A, then of B, each 2·planes KB.
    static __device__ __forceinline__ void load(const Operand& a, const Operand& b, int mb0, int nb0, int st,
                                                _Float16* stage, int wave, int lane) {
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
            const int i = wave + c * WAVES;  // wave-uniform
            if (i < MB) {
                const _Float16* g = a.data +
                                    ((size_t)min(mb0 + i, a.blocks - 1) * a.steps + 2 * st) * (PA * FRAG) + lane * 8;
                _Float16* l = stage + i * (2 * PA * FRAG);
                copy_to_lds<0>(g, l);
                copy_to_lds<1024>(g, l);
                if constexpr (PA == 2) {
                    copy_to_lds<2048>(g, l);
                    copy_to_lds<3072>(g, l);
                }
            } else {
                const _Float16* g = b.data + ((size_t)min(nb0 + i - MB, b.blocks - 1) * b.steps + 2 * st) * (PB * FRAG) +
                                    lane * 8;
                _Float16* l = stage + A_HALVES + (i - MB) * (2 * PB * FRAG);
                copy_to_lds<0>(g, l);
                copy_to_lds<1024>(g, l);
                if constexpr (PB == 2) {
                    copy_to_lds<2048>(g, l);
                    copy_to_lds<3072>(g, l);
                }
            }
        }
    }

    // One stage: B's fragments of a step once, A's a row block ahead. The scheduling barriers keep each group's reads
    // ahead of the products before it; left alone the compiler sinks them to their use, and every block waits for LDS.
    static __device__ __forceinline__ void multiply(const _Float16* stage, Acc& acc, int wm, int wn, int lane) {
        const _Float16* as = stage + wm * BM * (2 * PA * FRAG) + lane * 8;
        const _Float16* bs = stage + A_HALVES + wn * BN * (2 * PB * FRAG) + lane * 8;
        f16x8 a[2][PA], b[2][BN][PB];
        auto read_a = [&](int g) {
#pragma unroll
            for (int p = 0; p < PA; ++p)
                a[g & 1][p] = *reinterpret_cast<const f16x8*>(as + (((g % BM) * 2 + g / BM) * PA + p) * FRAG);
        };
        auto read_b = [&](int s) {
#pragma unroll
            for (int j = 0; j < BN; ++j)
#pragma unroll
                for (int p = 0; p < PB; ++p)
                    b[s][j][p] = *reinterpret_cast<const f16x8*>(bs + ((j * 2 + s) * PB + p) * FRAG);
        };
        read_b(0);
        read_a(0);
#pragma unroll
        for (int g = 0; g < 2 * BM; ++g) {
            const int s = g / BM, i = g % BM;
            if (g + 1 < 2 * BM) read_a(g + 1);
            if (g == (BM > 1 ? BM - 2 : 0)) read_b(1);
            __builtin_amdgcn_sched_barrier(0);
            // The pieces' products, smallest first.
#pragma unroll
            for (int j = 0; j < BN; ++j)
                if constexpr (PA == 2)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[g & 1][1], b[s][j][0], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < BN; ++j)
                if constexpr (PB == 2)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[g & 1][0], b[s][j][1], acc[i][j], 0, 0, 0);
#pragma unroll
            for (int j = 0; j < BN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[g & 1][0], b[s][j][0], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // acc = Σ over stages [s0, s1) of the tile at row blocks mb0 of A and nb0 of B. Every thread of the workgroup calls
    // it with the same arguments; it ends with the LDS free.
    static __device__ __forceinline__ void product(const Operand& a, const Operand& b, int mb0, int nb0, int s0, int s1,
                                                   _Float16* lds, Acc& acc, int wave, int lane) {
        const int wm = wave / WAVES_N, wn = wave % WAVES_N;
#pragma unroll
        for (int i = 0; i < BM; ++i)
#pragma unroll
            for (int j = 0; j < BN; ++j) acc[i][j] = f32x16{};
        if (s0 < s1) load(a, b, mb0, nb0, s0, lds, wave, lane);
        for (int st = s0; st < s1; ++st) {
            const int cur = (st - s0) & 1;
            // The stage's copies have landed, and every wave is done with the other buffer.
            __builtin_amdgcn_s_waitcnt(0);
            __builtin_amdgcn_s_barrier();
            if (st + 1 < s1) load(a, b, mb0, nb0, st + 1, lds + (cur ^ 1) * STAGE, wave, lane);
            multiply(lds + cur * STAGE, acc, wm, wn, lane);
        }
        __syncthreads();
    }
};

// A 32 x 32 block of outputs C[m, n] in one wave's accumulator: lane l holds column n = l mod 32, rows
// m = 8·(r / 4) + 4·(l / 32) + r mod 4. Written as fragments of Cᵀ (rows n, k = m): eight bytes a lane, each pair of
// lanes l, l + 32 filling a row's 16. `to`: the fragment pair's address for row block n / 32 and step m / 16.
__device__ __forceinline__ void store_transposed(const f32x16& c, _Float16* to, int lane) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        f16x4 hi, lo;
        split2h_4(f32x4{c[4 * q], c[4 * q + 1], c[4 * q + 2], c[4 * q + 3]}, 1.0f, hi, lo);
        _Float16* at = to + (q >> 1) * (2 * FRAG) + ((q & 1) * 32 + (lane & 31)) * 8 + 4 * (lane >> 5);
        *reinterpret_cast<f16x4*>(at) = hi;
        *reinterpret_cast<f16x4*>(at + FRAG) = lo;
    }
}

// The same block as fragments of C (rows m, k = n), turned in LDS: 32 rows of TURN dwords of the wave's own, each value
// as its two pieces in a dword. Rows 4 apart lie 32 banks apart (the two halves of a wave write without a conflict),
// and 8 consecutive rows' 16 bytes lie in different banks.
constexpr int TURN = 40, TURN_HALVES = 32 * TURN * 2;
__device__ __forceinline__ void turn_write(const f32x16& c, unsigned* turn, int lane) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        _Float16 hi, lo;
        split_value(c[r], hi, lo);
        turn[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * TURN + (lane & 31)] =
            (unsigned)__builtin_bit_cast(unsigned short, hi) | (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
    }
}
// Unit (row lane mod 32, columns 8·o … 8·o + 7) of the turned block, o = 2·pass + lane / 32.
__device__ __forceinline__ void turn_read(const unsigned* turn, int lane, int pass, f16x8& hi, f16x8& lo) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const unsigned* at = turn + (lane & 31) * TURN + (2 * pass + (lane >> 5)) * 8;
    const u32x4 x = *reinterpret_cast<const u32x4*>(at), y = *reinterpret_cast<const u32x4*>(at + 4);
    u32x4 h, l;
    h[0] = __builtin_amdgcn_perm(x[1], x[0], 0x05040100u);
    h[1] = __builtin_amdgcn_perm(x[3], x[2], 0x05040100u);
    h[2] = __builtin_amdgcn_perm(y[1], y[0], 0x05040100u);
    h[3] = __builtin_amdgcn_perm(y[3], y[2], 0x05040100u);
    l[0] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
    l[1] = __builtin_amdgcn_perm(x[3], x[2], 0x07060302u);
    l[2] = __builtin_amdgcn_perm(y[1], y[0], 0x07060302u);
    l[3] = __builtin_amdgcn_perm(y[3], y[2], 0x07060302u);
    hi = __builtin_bit_cast(f16x8, h);
    lo = __builtin_bit_cast(f16x8, l);
}

// The persistent workgroup's n-th unit: a round takes gridDim.x consecutive units, each XCD (workgroups are dealt to
// the 8 in turn) a run of them, so that units that share operands run on one XCD's L2. gridDim.x is a multiple of 8.
__device__ __forceinline__ int unit_of(int n) {
    return n * (int)gridDim.x + (int)(blockIdx.x & 7) * ((int)gridDim.x >> 3) + (int)(blockIdx.x >> 3);
}

}  // namespace packed
}  // namespace laya
