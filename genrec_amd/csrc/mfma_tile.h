// A 256 x BN tile of C[n][m] = sum_k A(m, k) B(n, k) on the matrix cores (v_mfma_f32_32x32x16_bf16, fp32
// accumulators), by one workgroup.  Both operands come through LDS by the copy path that bypasses the
// registers, 64 k at a time.  An operand lies in memory in one of four ways, each with a stage (what is copied where)
// and a reader (how a wave gets its fragments back):
//   MtAlong          rows of m (n), k along them
//   MtAcross         rows of k, m along them
//   MtBlocksAlong    blocks of 32 m (n) x 16 k in fragment order
//   MtBlocksAcross   such blocks made for the other axis: 32 k x 16 n
// An operand may lie in two bf16 pieces whose sum it is (16 bits of each element instead of 8): the pieces take turns as steps
// of k, and the other operand's k are taken twice.
// A fragment block is the 1 KB that one wave holds of a 32 x 16 operand: lane l has row l & 31, k = 8 (l >> 5) + 0 .. 7.
//
// C/D layout of the instruction: element e of lane l is m = (e & 3) + 8 (e >> 2) + 4 (l >> 5), n = l & 31: a lane
// holds one row n and runs of four m.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.h"

#define MT_BM 256
#define MT_BK 64

typedef short mt_s16x4 __attribute__((ext_vector_type(4)));
typedef short mt_s16x8 __attribute__((ext_vector_type(8)));
typedef float mt_f32x4 __attribute__((ext_vector_type(4)));
typedef float mt_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 mt_b16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mt_u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void mt_lds_void;
typedef __attribute__((address_space(3))) mt_s16x4 mt_lds_s16x4;
typedef __attribute__((address_space(3))) const mt_s16x8 mt_lds_s16x8;

// Waves as WM x WN, MA x NB blocks of 32 x 32 a wave.  DEEP, FLAT: buffers in LDS of the operand that comes from
// further away, and of the other one.
template <int BN>
struct MtShape;
template <> struct MtShape<256> { static constexpr int WM = 2, WN = 4, MA = 4, NB = 2, DEEP = 3, FLAT = 2, THREADS = 512; };
template <> struct MtShape<192> { static constexpr int WM = 4, WN = 2, MA = 2, NB = 3, DEEP = 3, FLAT = 2, THREADS = 512; };
template <> struct MtShape<128> { static constexpr int WM = 4, WN = 2, MA = 2, NB = 2, DEEP = 3, FLAT = 3, THREADS = 512; };
template <> struct MtShape<64> { static constexpr int WM = 8, WN = 1, MA = 1, NB = 2, DEEP = 2, FLAT = 2, THREADS = 512; };

template <int BN>
constexpr int mt_lds_bytes() {  // A is the deep one, or the two are alike
    return (MtShape<BN>::DEEP * MT_BM + MtShape<BN>::FLAT * BN) * MT_BK * 2;
}

__device__ __forceinline__ int mt_wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// The copy path from memory to LDS, 16 bytes a lane: from base + off (base uniform) or from a lane's own address to
// `to` (uniform) + 16 x lane.  As instructions of our own because the compiler, which cannot tell the buffers apart,
// puts a wait for all copies under way in front of every transposing LDS read; here they have no register result, and
// what has to be waited for is written out (mt_meet).  The compiler's own counts of loads under way come out too low
// beside them, which only makes its waits longer.  M0 is declared, so that nothing of the compiler's own is left in it across a
// copy; the warning that it is a register with a purpose of its own is expected.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void mt_copy(const char* base, uint32_t off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(to), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void mt_copy_from(const char* from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop

// ---- stages.  N: copies per wave and step (1 KB each); issue(i, to): the i-th of them into the buffer at
// `to`; advance(): on to the next step.  The addresses are a uniform base plus lane offsets that stay.  A copy writes
// lane l at 16 l, so the order inside a buffer is chosen by what each lane fetches: all orders below are such that no
// fragment read meets an LDS bank twice.

// Row r of a buffer: 64 k in 8 chunks of 16 bytes, chunk c at c ^ ((r >> 1) & 7).  Rows past the end read the last one:
// they make rows of C that nobody keeps.  Rows are less than 2^22 elements apart.
template <int W, int BN>
struct MtAlong {
    static constexpr int N = W * MT_BK * 2 / 16 / MtShape<BN>::THREADS;
    const char* base;
    uint32_t off[N];
    __device__ __forceinline__ MtAlong() {}
    __device__ __forceinline__ MtAlong(const uint16_t* p, int64_t ld, int rows, int at, int k0) {
        const int lane = threadIdx.x & 63, wave = mt_wave();
        base = reinterpret_cast<const char*>(p + (int64_t)at * ld + k0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int row = (wave * N + i) * 8 + (lane >> 3);
            const int chunk = (lane & 7) ^ ((row >> 1) & 7);
            row = at + row < rows ? row : rows - 1 - at;
            off[i] = (uint32_t)row * (uint32_t)ld * 2u + chunk * 16;
        }
    }
    __device__ __forceinline__ void issue(int i, uint32_t to) const { mt_copy(base, off[i], to + (mt_wave() * N + i) * 1024); }
    __device__ __forceinline__ void issue_any(int i, uint32_t to) const { issue(i, to); }
    __device__ __forceinline__ void advance() { base += MT_BK * 2; }
    __device__ __forceinline__ int whole_steps(int nk) const { return nk; }
};

// Row k of a buffer: 256 m in 32 chunks, chunk c at c ^ (4 (k & 3)).  Columns past the end (a multiple of 8) read the
// last eight; rows past the end read the last one, where the other operand is 0.  Every 64 k make two steps.
template <int BN>
struct MtAcross {
    static constexpr int N = 2048 / MtShape<BN>::THREADS;
    const char* base;
    uint32_t off[N];
    int64_t ld;
    int left;  // rows of k from the step's first on
    bool again;  // the step is the second one of its k
    __device__ __forceinline__ MtAcross() {}
    __device__ __forceinline__ MtAcross(const uint16_t* p, int64_t ld_, int cols, int k_rows, int at, int k0) {
        const int lane = threadIdx.x & 63, wave = mt_wave();
        ld = ld_;
        left = k_rows - k0;
        again = false;
        base = reinterpret_cast<const char*>(p + (int64_t)k0 * ld + at);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = (wave * N + i) * 2 + (lane >> 5);
            int col = ((lane & 31) ^ ((row & 3) << 2)) * 8;
            col = at + col < cols ? col : cols - 8 - at;
            off[i] = (uint32_t)row * (uint32_t)ld * 2u + (uint32_t)(col * 2);
        }
    }
    __device__ __forceinline__ void issue(int i, uint32_t to) const { mt_copy(base, off[i], to + (mt_wave() * N + i) * 1024); }
    __device__ __forceinline__ void issue_any(int i, uint32_t to) const {
        const int row = (mt_wave() * N + i) * 2 + ((threadIdx.x & 63) >> 5);
        const int64_t back = row < left ? 0 : (int64_t)(row - left + 1) * ld * 2;
        mt_copy_from(base + off[i] - back, to + (mt_wave() * N + i) * 1024);
    }
    __device__ __forceinline__ void advance() {
        base += again ? ld * (MT_BK * 2) : 0;
        left -= again ? MT_BK : 0;
        again = !again;
    }
    __device__ __forceinline__ int whole_steps(int nk) const {
        const int whole = left >= MT_BK ? left / MT_BK * 2 - (again ? 1 : 0) : 0;
        return nk < whole ? nk : whole;
    }
};

// W / 32 x 4 blocks a step: the four of a group of 32 rows in one piece, the groups of a pair one behind the other,
// pairs `pair_bytes` apart (less than 2^31 in all).  Groups past `groups` read the last one.  Odd steps stand `odd_bytes`
// behind even ones, those `even_bytes` behind odd ones.
template <int W, int BN>
struct MtBlocksAlong {
    static constexpr int N = W * MT_BK * 2 / 16 / MtShape<BN>::THREADS;
    const char* base;
    uint32_t off[N];
    int64_t step, then;
    __device__ __forceinline__ MtBlocksAlong() {}
    // p: the step's first block; groups: groups of 32 rows that are there from it on
    __device__ __forceinline__ MtBlocksAlong(const char* p, int64_t odd_bytes, int64_t even_bytes, uint32_t pair_bytes, int groups) {
        base = p;
        step = odd_bytes;
        then = even_bytes;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int block = mt_wave() * N + i;
            const int group = block / 4 < groups ? block / 4 : groups - 1;
            off[i] = (uint32_t)(group >> 1) * pair_bytes + ((group & 1) * 4 + block % 4) * 1024 + (threadIdx.x & 63) * 16;
        }
    }
    __device__ __forceinline__ void issue(int i, uint32_t to) const { mt_copy(base, off[i], to + (mt_wave() * N + i) * 1024); }
    __device__ __forceinline__ void issue_any(int i, uint32_t to) const { issue(i, to); }
    __device__ __forceinline__ void advance() {
        base += step;
        const int64_t s = step;
        step = then;
        then = s;
    }
    __device__ __forceinline__ int whole_steps(int nk) const { return nk; }
};

// G as d weight reads it: blocks of 32 n x 16 v, in memory [64 n][2 pieces][64 v][2][4], a step being one piece of 64 n of
// 256 v.
// In a buffer, [64 v][32 n][16 v] blocks whose unit of 16 bytes (n, 8 v h) stands at (2 n + h) ^ (8 in odd blocks): the
// 32 lanes of a transposing read take 16 different units of a bank row.
struct MtBlocksAcross {
    static constexpr int N = 2048 / MtShape<256>::THREADS;
    const char* base;
    uint32_t off[N];
    int64_t step;
    __device__ __forceinline__ MtBlocksAcross() {}
    __device__ __forceinline__ MtBlocksAcross(const char* p, int64_t step_bytes) {
        base = p;
        step = step_bytes;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int block = mt_wave() * N + i;
            const int unit = (threadIdx.x & 63) ^ ((block & 1) << 3);
            off[i] = block * 1024 + ((unit & 1) * 32 + (unit >> 1)) * 16;
        }
    }
    __device__ __forceinline__ void issue(int i, uint32_t to) const { mt_copy(base, off[i], to + (mt_wave() * N + i) * 1024); }
    __device__ __forceinline__ void issue_any(int i, uint32_t to) const { issue(i, to); }
    __device__ __forceinline__ void advance() { base += step; }
    __device__ __forceinline__ int whole_steps(int nk) const { return nk; }
};

// ---- readers: read(tile, sub, j) is fragment j (rows first + 32 j ...) of the 16 k at `sub` --------------------
struct MtReadAlong {
    uint32_t lane_off;
    __device__ __forceinline__ MtReadAlong(int first) {
        const int lane = threadIdx.x & 63, row = first + (lane & 31);
        lane_off = row * 128 + ((lane >> 5) ^ ((row >> 1) & 7)) * 16;
    }
    static constexpr int READS = 1;
    __device__ __forceinline__ mt_s16x8 read(uint32_t tile, int sub, int j) const {
        return *(mt_lds_s16x8*)(uintptr_t)(((tile + lane_off) ^ (sub * 32)) + j * 4096);
    }
};

// The transposing read works on 16 lanes: lane i fetches four m of row k + i / 4 and receives m = i of the four rows.
struct MtReadAcross {
    uint32_t lane_off;
    __device__ __forceinline__ MtReadAcross(int first) {
        const int i = threadIdx.x & 15, group = (threadIdx.x & 63) >> 4;
        const int k = (group >> 1) * 8 + (i >> 2), m = first + (group & 1) * 16 + (i & 3) * 4;
        lane_off = k * 512 + ((m >> 3) ^ ((k & 3) << 2)) * 16 + (m & 7) * 2;
    }
    static constexpr int READS = 2;
    __device__ __forceinline__ mt_s16x8 read(uint32_t tile, int sub, int j) const {
        const uint32_t q = ((tile + lane_off) ^ (j * 64)) + sub * 8192;
        const mt_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mt_lds_s16x4*)(uintptr_t)q);
        const mt_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mt_lds_s16x4*)(uintptr_t)(q + 2048));  // k + 4
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

struct MtReadBlocksAlong {
    uint32_t lane_off;
    __device__ __forceinline__ MtReadBlocksAlong(int first) { lane_off = (first >> 5) * 4096 + (threadIdx.x & 63) * 16; }
    static constexpr int READS = 1;
    __device__ __forceinline__ mt_s16x8 read(uint32_t tile, int sub, int j) const {
        return *(mt_lds_s16x8*)(uintptr_t)(tile + lane_off + j * 4096 + sub * 1024);
    }
};

struct MtReadBlocksAcross {
    uint32_t lane_off;
    __device__ __forceinline__ MtReadBlocksAcross(int first) {  // a multiple of 64
        const int i = threadIdx.x & 15, group = (threadIdx.x & 63) >> 4;
        const int unit = ((i >> 2) * 2 + ((i & 3) >> 1)) ^ ((group & 1) << 3);
        lane_off = (first >> 6) * 8192 + (group & 1) * 1024 + ((group >> 1) * 16 + unit) * 16 + (i & 1) * 8;
    }
    static constexpr int READS = 2;
    __device__ __forceinline__ mt_s16x8 read(uint32_t tile, int sub, int j) const {
        const uint32_t q = tile + lane_off, at = (sub >> 1) * 4096 + (sub & 1) * 512 + j * 2048;
        const mt_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mt_lds_s16x4*)(uintptr_t)(q + at));
        const mt_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mt_lds_s16x4*)(uintptr_t)((q ^ 128) + at));  // n + 4
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// ---- the pipeline ------------------------------------------------------------------------------------------
// Waits until at most VM of this wave's copies are under way and its LDS reads are done, then meets the other waves.
template <int VM>
__device__ __forceinline__ void mt_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(VM) : "memory");
}

// begin() starts the first copies of a tile (the LDS must be free), run() adds the products to acc and leaves the LDS
// free: the next
// tile's begin() may come before this one's results are used, so that its copies travel meanwhile.
//
// One meeting of the waves per step, in front of its last quarter: by then every wave holds that quarter's fragments
// in registers, so the step's buffers are free for the copies of a later step, and the next step's copies, under way
// for one or two steps, have landed -- its first fragments are read between the products of the last quarter.
// Every LDS read goes out a quarter before its product, early in it, and the copies of a step are spread over two
// quarters, one behind a product: nothing in the loop waits for what was issued right before.
template <int BN, class StageA, class ReadA, class StageB, class ReadB, bool B_DEEP = false, int DEEP = MtShape<BN>::DEEP>
struct MtPipe {
    typedef MtShape<BN> S;
    static constexpr int AR = B_DEEP ? S::FLAT : DEEP, BR = B_DEEP ? DEEP : S::FLAT;
    typedef mt_f32x16 Acc[S::MA][S::NB];
    static constexpr int A_BYTES = MT_BM * MT_BK * 2, B_BYTES = BN * MT_BK * 2;
    StageA sa;
    StageB sb;
    int nk;
    uint32_t la, lb;

    __device__ __forceinline__ explicit MtPipe(unsigned char* lds) {
        la = (uint32_t)(uintptr_t)(mt_lds_void*)lds;
        lb = la + AR * A_BYTES;
    }
    __device__ __forceinline__ void begin(const StageA& a, const StageB& b, int steps) {
        sa = a;
        sb = b;
        nk = steps;
#pragma unroll
        for (int t = 0; t < DEEP; ++t) {
            if (t < BR && t < nk) {
#pragma unroll
                for (int i = 0; i < StageB::N; ++i) sb.issue_any(i, lb + t * B_BYTES);
                sb.advance();
            }
            if (t < AR && t < nk) {
#pragma unroll
                for (int i = 0; i < StageA::N; ++i) sa.issue_any(i, la + t * A_BYTES);
                sa.advance();
            }
        }
    }
    static __device__ __forceinline__ void clear(Acc& acc) {
#pragma unroll
        for (int m = 0; m < S::MA; ++m)
#pragma unroll
            for (int n = 0; n < S::NB; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.f;
    }
    // The 32 elements of block m of a lane's row n from memory (p: the row at the block), as they lie in acc.
    static __device__ __forceinline__ void load(Acc& acc, int m, int n, const float* p) {
        const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const mt_f32x4 v = *reinterpret_cast<const mt_f32x4*>(p + 8 * q + 4 * half);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[m][n][4 * q + j] = v[j];
        }
    }
    // stores: at least LATER vector memory instructions of this wave came behind begin()'s copies (stores of the tile
    // before); they need not have ended.  Memory instructions of a wave end in their order on this target.
    template <int LATER = 0>
    __device__ __forceinline__ void run(Acc& acc, bool stores = false) {
        if (nk <= 0) return;
        const int wave = mt_wave();
        const ReadA ra(wave / S::WN * S::MA * 32);
        const ReadB rb(wave % S::WN * S::NB * 32);
        constexpr int AHEAD = (AR - 2) * StageA::N + (BR - 2) * StageB::N;  // copies that may stay under way
        if (LATER > 0 && stores) mt_meet<LATER>();
        else mt_meet<0>();
        uint32_t ca = la, cb = lb;  // the present step's buffers
        mt_s16x8 fa[2][S::MA], fb[2][S::NB];
#pragma unroll
        for (int j = 0; j < S::NB; ++j) fb[0][j] = rb.read(cb, 0, j);
#pragma unroll
        for (int j = 0; j < S::MA; ++j) fa[0][j] = ra.read(ca, 0, j);

        // the products of fragment set `set`, with the reads of (ra_at, rb_at, sub) into the other set and `n` copies
        // (copy(i)) between them
        auto quarter = [&](auto set_, uint32_t ra_at, uint32_t rb_at, int sub, auto n_, auto&& copy) {
            constexpr int set = decltype(set_)::value, COPIES = decltype(n_)::value;
            constexpr int FRAGS = S::MA + S::NB, PRODUCTS = S::MA * S::NB;
            constexpr int PER = (2 * FRAGS + PRODUCTS - 1) / PRODUCTS;  // all reads in the first half of the products
#pragma unroll
            for (int p = 0; p < PRODUCTS; ++p) {
                __builtin_amdgcn_sched_barrier(0);
                const int m = p / S::NB, n = p % S::NB;
                acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[set][m], fb[set][n], acc[m][n], 0, 0, 0);
#pragma unroll
                for (int f = p * PER; f < (p + 1) * PER; ++f) {
                    if (f < S::NB) fb[set ^ 1][f] = rb.read(rb_at, sub, f);
                    else if (f < FRAGS) fa[set ^ 1][f - S::NB] = ra.read(ra_at, sub, f - S::NB);
                }
#pragma unroll
                for (int i = p * COPIES / PRODUCTS; i < (p + 1) * COPIES / PRODUCTS; ++i) copy(i);
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        typedef std::integral_constant<int, 0> Zero;
        typedef std::integral_constant<int, 1> One;
        auto none = [](int) {};
        int ia = 0, ib = 0, kt = 0;
        uint32_t free_deep = 0;
        // Copies in step kt: the deep operand's of step kt - 1 + its depth in the first quarter, the flat one's of step
        // kt + its depth in the last, so that what is needed first goes out first.
        auto step = [&](auto whole_, bool deep_due) {
            constexpr bool whole = decltype(whole_)::value;
            if constexpr (whole) {
                if constexpr (B_DEEP) {
                    quarter(Zero(), ca, cb, 1, std::integral_constant<int, StageB::N>(), [&](int i) { sb.issue(i, free_deep); });
                    sb.advance();
                } else {
                    quarter(Zero(), ca, cb, 1, std::integral_constant<int, StageA::N>(), [&](int i) { sa.issue(i, free_deep); });
                    sa.advance();
                }
            } else {
                quarter(Zero(), ca, cb, 1, Zero(), none);
                if (deep_due) {
                    if constexpr (B_DEEP) {
#pragma unroll
                        for (int i = 0; i < StageB::N; ++i) sb.issue_any(i, free_deep);
                        sb.advance();
                    } else {
#pragma unroll
                        for (int i = 0; i < StageA::N; ++i) sa.issue_any(i, free_deep);
                        sa.advance();
                    }
                }
            }
            quarter(One(), ca, cb, 2, Zero(), none);
            quarter(Zero(), ca, cb, 3, Zero(), none);
            if (whole) mt_meet<AHEAD>();
            else mt_meet<0>();
            const uint32_t free_flat = B_DEEP ? ca : cb;
            free_deep = B_DEEP ? cb : ca;
            ia = ia + 1 == AR ? 0 : ia + 1;
            ib = ib + 1 == BR ? 0 : ib + 1;
            ca = la + ia * A_BYTES;
            cb = lb + ib * B_BYTES;
            if constexpr (whole) {
                if constexpr (B_DEEP) {
                    quarter(One(), ca, cb, 0, std::integral_constant<int, StageA::N>(), [&](int i) { sa.issue(i, free_flat); });
                    sa.advance();
                } else {
                    quarter(One(), ca, cb, 0, std::integral_constant<int, StageB::N>(), [&](int i) { sb.issue(i, free_flat); });
                    sb.advance();
                }
            } else {
                if (kt + S::FLAT < nk) {
                    if constexpr (B_DEEP) {
#pragma unroll
                        for (int i = 0; i < StageA::N; ++i) sa.issue_any(i, free_flat);
                        sa.advance();
                    } else {
#pragma unroll
                        for (int i = 0; i < StageB::N; ++i) sb.issue_any(i, free_flat);
                        sb.advance();
                    }
                }
                // behind the last step: whatever the next buffer holds, not used
                quarter(One(), ca, cb, 0, Zero(), none);
            }
        };
        // whole steps of either operand, as seen behind the copies of begin()
        const int wa = sa.whole_steps(nk - AR) + AR, wb = sb.whole_steps(nk - BR) + BR;
        const int wd = (B_DEEP ? wb : wa) - DEEP + 1, wf = (B_DEEP ? wa : wb) - S::FLAT;
        const int safe = wd < wf ? wd : wf;
        step(std::false_type(), false);
        for (kt = 1; kt < safe; ++kt) step(std::true_type(), true);
        for (; kt < nk; ++kt) step(std::false_type(), kt - 1 + DEEP < nk);
        mt_meet<0>();
    }
};

// Workgroups are dealt to the eight XCDs round robin, and about 32 run on each at a time.  All XCDs work on the same
// few m tiles at a time -- the large operand, which one of them fetches from memory and the others from the cache
// behind the L2s -- and each keeps to its own n tiles (n tile = XCD modulo 8) where there are that many; else
// an m tile stays on one XCD with all its n tiles.
__device__ __forceinline__ void mt_tile(int block, int m_tiles, int n_tiles, int& tm, int& tn) {
    if (n_tiles >= 8) {
        tm = block / n_tiles;
        tn = block - tm * n_tiles;
        return;
    }
    const int group = block / (8 * n_tiles), left = m_tiles - group * 8;
    const int rest = block - group * 8 * n_tiles, wide = left < 8 ? left : 8;
    tn = rest / wide;
    tm = group * 8 + rest - tn * wide;
}

// Eight m of a lane's row in memory order: quads 2 q and 2 q + 1 of a 32 x 32 block (elements 8 q ..), rounded to bf16,
// as the half of the wave that holds m 16 q + 8 (l >> 5) + 0 .. 7.  The halves trade their middle runs of four.
__device__ __forceinline__ mt_u32x4 mt_pack8(mt_f32x4 x, mt_f32x4 y) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 a = __builtin_bit_cast(u2, __builtin_convertvector(x, mt_b16x4));
    const u2 b = __builtin_bit_cast(u2, __builtin_convertvector(y, mt_b16x4));
    const auto p = __builtin_amdgcn_permlane32_swap(a.x, b.x, false, false);
    const auto q = __builtin_amdgcn_permlane32_swap(a.y, b.y, false, false);
    return mt_u32x4{p[0], q[0], p[1], q[1]};
}

// What rounding to bf16 takes from x: the second piece.
__device__ __forceinline__ mt_f32x4 mt_rest(mt_f32x4 x) {
    return x - __builtin_convertvector(__builtin_convertvector(x, mt_b16x4), mt_f32x4);
}

// Two blocks of results (m rows of 32 and the next 32, 32 n) rounded to bf16 and stored as 32 rows n of 64 m.
// Through 4 KB of LDS that belong to this wave (at `lds`, a byte address), in whole lines of 128 bytes.  out: the first
// row's first element; row r is written if r < rows.
__device__ __forceinline__ void mt_store_rows(const mt_f32x16& c0, const mt_f32x16& c1, uint32_t lds, uint16_t* out, int64_t ld, int rows) {
    typedef __attribute__((address_space(3))) mt_u32x4 lds_u32x4;
    const int lane = threadIdx.x & 63, row = lane & 31;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const mt_f32x16& c = k < 2 ? c0 : c1;
        const int q = 8 * (k & 1), chunk = k * 2 + (lane >> 5);
        const mt_f32x4 x = {c[q], c[q + 1], c[q + 2], c[q + 3]}, y = {c[q + 4], c[q + 5], c[q + 6], c[q + 7]};
        *(lds_u32x4*)(uintptr_t)(lds + row * 128 + ((chunk ^ (row & 7)) << 4)) = mt_pack8(x, y);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 3), chunk = lane & 7;
        const mt_u32x4 v = *(lds_u32x4*)(uintptr_t)(lds + r * 128 + ((chunk ^ (r & 7)) << 4));
        if (r < rows) __builtin_nontemporal_store(v, reinterpret_cast<mt_u32x4*>(out + r * ld + chunk * 8));
    }
}

// The same from the registers, 16 bytes a lane.  out: the first element of this lane's row.
__device__ __forceinline__ void mt_store_lanes(const mt_f32x16& c0, const mt_f32x16& c1, uint16_t* out) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const mt_f32x16& c = k < 2 ? c0 : c1;
        const int q = 8 * (k & 1);
        const mt_f32x4 x = {c[q], c[q + 1], c[q + 2], c[q + 3]}, y = {c[q + 4], c[q + 5], c[q + 6], c[q + 7]};
        *reinterpret_cast<mt_u32x4*>(out + 16 * k + 8 * half) = mt_pack8(x, y);
    }
}
