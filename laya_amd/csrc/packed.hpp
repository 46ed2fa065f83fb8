// Products of packed operands: the matrix-core loop of the vocabulary cross entropy (vocab.hip) and the Newton-Schulz
// iteration (muon.hip).
//
// An fp32 operand that several tiles read is split once into the fp16 pieces of split2h_4 (a power-of-two scale, then
// hi + lo, 22 bits) and kept in the order in which the matrix cores take it, so that the product's loop converts
// nothing and computes no addresses: it copies runs of memory to LDS (16 bytes a lane, no registers between) and reads
// fragments back, both linear. v_mfma_f32_16x16x32_f16 takes from lane l the 8 k of l / 16 of row l mod 16, so a
// fragment is 16 rows x 32 k = 1 KB, [k / 8][row][8 k], and an operand of R rows and K columns is
//   [⌈R / 32⌉ row groups][⌈K / 32⌉ steps][2 halves of 16 rows][planes: hi, lo][512 fp16]
// with zeros behind R and K. bf16-valued operands keep one plane (split1h_4). Three piece products make one
// fp32-accurate product (lo·hi, hi·lo, hi·hi), two when one side has one plane.
//
// The same memory serves a product over the operand's rows (its columns then being the product's rows): a row group's
// step is 32 x 32 values either way, and ds_read_b64_tr_b16 hands each lane four rows of its column. Octet o's rows
// stand rotated by 4·o, so that the four rows x two octets that such a read meets lie in different banks; a linear read
// takes each lane's unit through the same rotation, still 1 KB in a row.
//
// These products are bound by the power that the matrix cores draw, not by their rate: on random fp16 data (registers
// and LDS alone) 16x16x32 reaches 1.81 PFLOP/s and 32x32x16 1.59, on zeros both 2.38. Hence the 16 x 16 form.
#pragma once
#include <type_traits>

#include "common.hpp"
#include "split.hpp"

namespace laya {
namespace packed {

constexpr int FRAG = 512;  // fp16 values of a fragment

inline int groups_of(long rows) { return (int)((rows + 31) / 32); }
inline int steps_of(long k) { return (int)((k + 31) / 32); }
inline size_t halves(long rows, long k, int planes) { return (size_t)groups_of(rows) * steps_of(k) * 2 * planes * FRAG; }

// A packed operand as a kernel takes it. `groups`: its row groups (a tile's groups behind the last read the last).
struct Operand {
    const _Float16* data;
    int steps, groups;
};

// Where the hi plane's 8 values of row r, columns 8·o …, of a row group's step start (o: the octet of the 32 columns).
template <int PLANES>
__device__ __forceinline__ int unit_at(int r, int o) {
    return ((r >> 4) * PLANES * 4 + o) * 128 + ((r + 4 * o) & 15) * 8;
}

__device__ __forceinline__ void split_value(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// KB KB from global memory to LDS, 16 bytes a lane and KB, the wave's 64 lanes in a row from LDS byte `to` (the same in
// every lane). Written as assembly, which takes no register for the data: around the builtin the compiler lets every
// LDS read wait for all reads before it (it cannot tell the copy's target from theirs), and the loop's look-ahead is
// lost. The loop waits for the copies itself (wait_copies).
template <int KB>
__device__ __forceinline__ void copy_to_lds(const _Float16* from, unsigned to) {
    static_assert(KB == 2 || KB == 4, "a row group's step");
    constexpr int KIB = 1024;
    if constexpr (KB == 4)
        asm volatile(
            "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t"
            "global_load_lds_dwordx4 %1, off offset:%2\n\tglobal_load_lds_dwordx4 %1, off offset:%3\n\t"
            "global_load_lds_dwordx4 %1, off offset:%4" ::"s"(to), "v"(from), "n"(KIB), "n"(2 * KIB), "n"(3 * KIB) : "memory");
    else
        asm volatile(
            "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t"
            "global_load_lds_dwordx4 %1, off offset:%2" ::"s"(to), "v"(from), "n"(KIB) : "memory");
}
// Waits for all but the wave's last N copies (and its other memory accesses before them), then for the whole workgroup:
// what every wave copied before its last N is in LDS, and every wave's reads before this point are done.
template <int N>
__device__ __forceinline__ void wait_copies() {
    static_assert(N < 64, "vmcnt");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
__device__ __forceinline__ unsigned lds_byte(const void* p) {
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// One side's fragments as a wave reads them from a step in LDS. T: the operand's columns are the product's rows.
template <int PLANES, bool T>
struct Reader {
    const _Float16* at[T ? 4 : 1];  // T: [16-column half][rows 4·p … 4·p + 3 of the lane's octet of rows]
    __device__ __forceinline__ Reader(const _Float16* side, int lane) {
        if constexpr (T) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = 8 * (lane >> 4) + 4 * (q & 1) + ((lane & 15) >> 2), c = lane & 3;
                at[q] = side + unit_at<PLANES>(r, 2 * (q >> 1) + (c >> 1)) + 4 * (c & 1);
            }
        } else {
            at[0] = side + unit_at<PLANES>(lane & 15, lane >> 4);
        }
    }
    // Block i (16 of the product's rows), plane p, of the step `step` halves into the side's memory.
    __device__ __forceinline__ f16x8 read(int step, int i, int p) const {
        if constexpr (T) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            const int o = step + (i >> 1) * (2 * PLANES * FRAG) + p * FRAG;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(at[2 * (i & 1)] + o));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(at[2 * (i & 1) + 1] + o));
            return __builtin_shufflevector(__builtin_bit_cast(f16x4, lo), __builtin_bit_cast(f16x4, hi), 0, 1, 2, 3, 4,
                                           5, 6, 7);
        } else {
            return *reinterpret_cast<const f16x8*>(at[0] + step + (i * PLANES + p) * FRAG);
        }
    }
};

// A workgroup of WAVES_M x WAVES_N waves, each BM x BN blocks of 16 x 16 outputs: C[m, n] += Σ_k A[m, k]·B[n, k]. TA, TB:
// that side is packed with the product's k as its rows.
//
// LDS holds a ring of 32-deep steps. A step's barrier stands before its last row block's products: by then every wave has
// read the step to the end and the next step's copies, started RING − 1 steps ago, have landed; behind it the copies of
// the step RING ahead start into the buffer just read, and the next step's first fragments are read while the last
// products run. Between two barriers a wave has a whole step's products, and no read or copy is waited for where it is
// issued. Two steps fill LDS with 256 x 256 tiles (and a step is long enough for a copy); small tiles, whose steps are
// shorter than a copy takes, look further ahead.
template <int WAVES_M, int WAVES_N, int BM, int BN, int PA, int PB, bool TA = false, bool TB = false, int RING = 2>
struct Tile {
    static constexpr int WAVES = WAVES_M * WAVES_N, THREADS = 64 * WAVES;
    static constexpr int M = WAVES_M * BM * 16, N = WAVES_N * BN * 16;
    static constexpr int MG = M / 32, NG = N / 32;  // row groups of A and B in a tile
    static constexpr int A_HALVES = MG * 2 * PA * FRAG, STEP = A_HALVES + NG * 2 * PB * FRAG;
    static constexpr int LDS_HALVES = RING * STEP;
    static constexpr int PER_WAVE = (MG + NG) / WAVES;  // row groups a wave copies each step
    static_assert((MG + NG) % WAVES == 0 && PER_WAVE <= 2 && BM % 2 == 0 && BN % 2 == 0 &&
                      (MG % WAVES == 0 || PA == PB), "tile shape");

    static constexpr int COPIES = MG % WAVES == 0 ? MG / WAVES * 2 * PA + NG / WAVES * 2 * PB : PER_WAVE * 2 * PA;

    typedef f32x4 Acc[BM][BN];

    // Planes of the c-th row group that a wave copies (A's come first).
    static constexpr int planes(int c) { return MG % WAVES == 0 ? (c < MG / WAVES ? PA : PB) : PA; }

    struct Copies {
        const _Float16* from[PER_WAVE];
        size_t next[PER_WAVE];  // from a step to the next
        unsigned to[PER_WAVE];
        // Starts a step's copies into the buffer at byte `slot`, and moves on to the next step.
        __device__ __forceinline__ void start(unsigned slot) {
            copy<0>(slot);
            if constexpr (PER_WAVE > 1) copy<1>(slot);
        }
        template <int C>
        __device__ __forceinline__ void copy(unsigned slot) {
            copy_to_lds<2 * planes(C)>(from[C], to[C] + slot);
            from[C] += next[C];
        }
    };

    typedef Reader<PA, TA> ReadA;
    typedef Reader<PB, TB> ReadB;
    static __device__ __forceinline__ void read_a(const ReadA& as, int step, int i, f16x8 (&a)[PA]) {
#pragma unroll
        for (int p = 0; p < PA; ++p) a[p] = as.read(step, i, p);
    }
    static __device__ __forceinline__ void read_b(const ReadB& bs, int step, int j, f16x8 (&b)[PB]) {
#pragma unroll
        for (int p = 0; p < PB; ++p) b[p] = bs.read(step, j, p);
    }
    // The pieces' products, smallest first: of a whole row block, piece by piece (no product waits for the one before),
    // and of one block.
    static __device__ __forceinline__ void mma(const f16x8 (&a)[PA], const f16x8 (&b)[BN][PB], f32x4 (&c)[BN]) {
        if constexpr (PA == 2)
#pragma unroll
            for (int j = 0; j < BN; ++j) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], b[j][0], c[j], 0, 0, 0);
        if constexpr (PB == 2)
#pragma unroll
            for (int j = 0; j < BN; ++j) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[j][1], c[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < BN; ++j) c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[j][0], c[j], 0, 0, 0);
    }
    static __device__ __forceinline__ void mma1(const f16x8 (&a)[PA], const f16x8 (&b)[PB], f32x4& c) {
        if constexpr (PA == 2) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], b[0], c, 0, 0, 0);
        if constexpr (PB == 2) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[0], c, 0, 0, 0);
    }

    // acc = Σ over steps [s0, s1) of the tile at row groups mg0 of A and ng0 of B. Every thread of the workgroup calls it
    // with the same arguments; it ends with the LDS free.
    static __device__ __forceinline__ void product(const Operand& a, const Operand& b, int mg0, int ng0, int s0, int s1,
                                                   _Float16* lds, Acc& acc, int wave, int lane) {
        const int wm = wave / WAVES_N, wn = wave % WAVES_N;
#pragma unroll
        for (int i = 0; i < BM; ++i)
#pragma unroll
            for (int j = 0; j < BN; ++j) acc[i][j] = f32x4{};
        if (s0 >= s1) return;
        Copies cp;
        const unsigned lds0 = lds_byte(lds);
#pragma unroll
        for (int c = 0; c < PER_WAVE; ++c) {
            const int i = __builtin_amdgcn_readfirstlane(wave + c * WAVES);
            const bool on_a = i < MG, turned = on_a ? TA : TB;
            const Operand& o = on_a ? a : b;
            const int at = on_a ? mg0 + i : ng0 + i - MG, size = 2 * (on_a ? PA : PB) * FRAG;
            cp.from[c] = o.data + lane * 8 +
                         (turned ? (size_t)s0 * o.steps + min(at, o.steps - 1)
                                 : (size_t)min(at, o.groups - 1) * o.steps + s0) * size;
            cp.next[c] = (turned ? (size_t)o.steps : (size_t)1) * size;
            cp.to[c] = lds0 + 2 * (on_a ? i * size : A_HALVES + (i - MG) * size);
        }
        const ReadA as(lds + wm * BM * (PA * FRAG), lane);
        const ReadB bs(lds + A_HALVES + wn * BN * (PB * FRAG), lane);
        const int len = s1 - s0;
#pragma unroll
        for (int q = 0; q < RING; ++q)
            if (q < len) cp.start(q * (2 * STEP));
        if (len >= RING)
            wait_copies<(RING - 1) * COPIES>();
        else
            wait_copies<0>();
        f16x8 fa[2][PA], fb[BN][PB];
        read_a(as, 0, 0, fa[0]);
#pragma unroll
        for (int j = 0; j < BN; ++j) read_b(bs, 0, j, fb[j]);
        // One step from the buffer at `at` (its fragments of B in fb, A's first in fa[0]); the last row block's products hand
        // fb over to the next step's, block by block. `ahead`: the steps behind it. What is read ahead of the last step's
        // end is of a buffer that no one needs.
        auto step = [&](int at, int next, int ahead) {
#pragma unroll
            for (int i = 0; i + 1 < BM; ++i) {
                read_a(as, at, i + 1, fa[(i + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
                mma(fa[i & 1], fb, acc[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (RING == 2 || ahead < RING)
                wait_copies<0>();
            else
                wait_copies<(RING - 2) * COPIES>();
            if (ahead >= RING) cp.start(2 * at);
            read_a(as, next, 0, fa[0]);
#pragma unroll
            for (int j = 0; j < BN; ++j) {
                mma1(fa[1], fb[j], acc[BM - 1][j]);
                __builtin_amdgcn_sched_barrier(0);
                read_b(bs, next, j, fb[j]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        int left = len;
        if constexpr (RING == 2) {
            for (; left > 1; left -= 2) {
                step(0, STEP, left - 1);
                step(STEP, 0, left - 2);
            }
            if (left > 0) step(0, STEP, 0);
        } else {
            for (int at = 0; left > 0; --left) {
                const int next = at + STEP == RING * STEP ? 0 : at + STEP;
                step(at, next, left - 1);
                at = next;
            }
        }
        __syncthreads();
    }
};

// 32 x 32 outputs C[m, n] as two by two blocks of one wave's accumulator: lane l holds column n = l mod 16 of a block,
// rows m = 4·(l / 16) … + 3.

// Written as a row group's step of Cᵀ (rows n, k = m), eight bytes a lane.
__device__ __forceinline__ void store_transposed(const f32x4 (&c)[2][2], _Float16* to, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f16x4 hi, lo;
            split2h_4(c[i][j], 1.0f, hi, lo);
            _Float16* at = to + unit_at<2>(16 * j + (lane & 15), 2 * i + (lane >> 5)) + 4 * ((lane >> 4) & 1);
            *reinterpret_cast<f16x4*>(at) = hi;
            *reinterpret_cast<f16x4*>(at + FRAG) = lo;
        }
}

// The same outputs turned in LDS to a row group's step of C (rows m, k = n): 32 rows of TURN dwords of the wave's own,
// each value as its two pieces in a dword. The rows that a write's four quarters meet lie 16 banks apart, and 16
// consecutive rows' 16 bytes in different banks.
constexpr int TURN = 36, TURN_DWORDS = 32 * TURN;
__device__ __forceinline__ void turn_write(const f32x4 (&c)[2][2], unsigned* turn, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                _Float16 hi, lo;
                split_value(c[i][j][r], hi, lo);
                turn[(16 * i + 4 * (lane >> 4) + r) * TURN + 16 * j + (lane & 15)] =
                    (unsigned)__builtin_bit_cast(unsigned short, hi) |
                    (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
            }
}
// The lane's unit of row half i: row 16·i + l mod 16, columns 8·(l / 16) … + 7.
__device__ __forceinline__ void turn_read(const unsigned* turn, int lane, int i, f16x8& hi, f16x8& lo) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const unsigned* at = turn + (16 * i + (lane & 15)) * TURN + (lane >> 4) * 8;
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
