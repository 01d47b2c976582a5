// A 256 x BN tile of C[n][m] = sum_k A(m, k) B(n, k) on the matrix cores (v_mfma_f32_32x32x16_bf16, fp32
// accumulators), by one workgroup of eight waves.  Either operand lies in memory with k running along its rows
// (rows of m or n) or across them (rows of k); both come through LDS by the copy path that bypasses the registers,
// two tiles of 64 k in turn, so that the next one travels while the present one is multiplied.
//
// C/D layout of the instruction: element e of lane l is m = (e & 3) + 8 (e >> 2) + 4 (l >> 5), n = l & 31: a lane
// holds one row n and runs of four m.
#pragma once

#include <hip/hip_runtime.h>

#include "common.h"

#define MT_THREADS 512
#define MT_BM 256
#define MT_BK 64

typedef short mt_s16x4 __attribute__((ext_vector_type(4)));
typedef short mt_s16x8 __attribute__((ext_vector_type(8)));
typedef float mt_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 mt_b16x4 __attribute__((ext_vector_type(4)));
typedef float mt_f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void mt_lds_void;
typedef __attribute__((address_space(3))) mt_s16x4 mt_lds_s16x4;
typedef __attribute__((address_space(1))) const void mt_global_void;

// One operand: `rows` rows of `ld` elements.  k along: a row per m (n), starting at column k0; rows past the end
// read the last one, and k0 + 64 nk elements of each are there.  k across: a row per k, starting at row k0, columns
// past the end (a multiple of 8) read the last eight, rows past the end the last row: the other operand is 0 there.
// What else is read twice is multiplied into elements of C that nobody keeps.
struct MtOperand {
    const uint16_t* p;
    int64_t ld;
    int extent;  // valid m (n)
    int k_rows;  // k across: rows of k
};

template <int BN>
struct MtShape;  // waves as WM x WN, MA x NB blocks of 32 x 32 a wave
template <> struct MtShape<256> { static constexpr int WM = 2, WN = 4, MA = 4, NB = 2; };
template <> struct MtShape<128> { static constexpr int WM = 4, WN = 2, MA = 2, NB = 2; };
template <> struct MtShape<64> { static constexpr int WM = 8, WN = 1, MA = 1, NB = 2; };

template <int BN>
constexpr int mt_lds_bytes() { return 2 * (MT_BM + BN) * MT_BK * 2; }

// LDS images, in chunks of 16 bytes, permuted so that no read meets a bank twice:
//  k along:  row r holds 64 k (8 chunks), chunk c at c ^ ((r >> 1) & 7): the 16 lanes that read the same chunk of
//            consecutive rows find 16 different chunks of a 256-byte bank row (two rows).
//  k across: row k holds W elements, chunk c at c ^ (4 (k & 3)): 32 lanes of a transposing read take four chunks of
//            each of four rows.
// The copy writes lane l of an instruction at base + 16 l, so the permutation is applied to the source address.
__device__ __forceinline__ int mt_swz_along(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }
__device__ __forceinline__ int mt_swz_across(int k, int chunk) { return chunk ^ ((k & 3) << 2); }

// W: rows (k along) or columns (k across) of the operand's tile
template <int W, bool ACROSS>
struct MtStage {
    static constexpr int N = W * MT_BK * 2 / 1024 / 8;  // instructions per wave: 1 KB each, eight waves
    const uint16_t* src[N];
    int64_t ld;
    int k[N], k_last;
    __device__ __forceinline__ MtStage(const MtOperand& o, int at, int k0) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (ACROSS) {
                constexpr int PER = 64 / (W / 8);  // rows of k per instruction
                const int row = (wave * N + i) * PER + lane / (W / 8);
                int col = at + mt_swz_across(row, lane % (W / 8)) * 8;
                col = col < o.extent ? col : o.extent - 8;
                src[i] = o.p + col;
                k[i] = k0 + row;
            } else {
                const int r = (wave * N + i) * 8 + (lane >> 3);
                int row = at + r;
                row = row < o.extent ? row : o.extent - 1;
                src[i] = o.p + (int64_t)row * o.ld + k0 + mt_swz_along(r, lane & 7) * 8;
            }
        }
        ld = o.ld;
        k_last = o.k_rows - 1;
    }
    __device__ __forceinline__ void issue(unsigned char* dst) {
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint16_t* from = src[i];
            if (ACROSS) {
                from += (int64_t)(k[i] < k_last ? k[i] : k_last) * ld;
                k[i] += MT_BK;
            } else {
                src[i] += MT_BK;
            }
            __builtin_amdgcn_global_load_lds((mt_global_void*)from, (mt_lds_void*)(dst + (wave * N + i) * 1024), 16, 0, 0);
        }
    }
};

// The fragment of the 32 x 16 block at row `at` (inside the tile) and sub-step `sub`: lane l gets row l & 31,
// k = 8 (l >> 5) + 0 .. 7.
template <int W, bool ACROSS>
__device__ __forceinline__ mt_s16x8 mt_fragment(const unsigned char* tile, int at, int sub) {
    const int lane = threadIdx.x & 63;
    if constexpr (!ACROSS) {
        const int row = at + (lane & 31);
        return *reinterpret_cast<const mt_s16x8*>(tile + row * 128 + mt_swz_along(row, 2 * sub + (lane >> 5)) * 16);
    } else {
        // the transposing read works on 16 lanes: lane i fetches four m of row k + i / 4 and receives element m = i of
        // the four rows
        const int i = lane & 15, group = lane >> 4;
        const int k = sub * 16 + (group >> 1) * 8 + (i >> 2);
        const int m = at + (group & 1) * 16 + (i & 3) * 4;
        const unsigned char* p = tile + k * (W * 2) + mt_swz_across(k, m >> 3) * 16 + (m & 7) * 2;
        const mt_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mt_lds_s16x4*)p);
        const mt_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((mt_lds_s16x4*)(p + 4 * (W * 2)));  // k + 4: same permutation
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// acc += over nk steps of 64 k.  Ends with a barrier: the LDS is free again.
template <int BN, bool A_ACROSS, bool B_ACROSS>
__device__ __forceinline__ void mt_multiply(mt_f32x16 (&acc)[MtShape<BN>::MA][MtShape<BN>::NB], unsigned char* lds,
                                            const MtOperand& a, int m0, const MtOperand& b, int n0, int k0, int nk) {
    typedef MtShape<BN> S;
    constexpr int A_BYTES = MT_BM * MT_BK * 2, BUF = A_BYTES + BN * MT_BK * 2;
    const int wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN;
    MtStage<MT_BM, A_ACROSS> sa(a, m0, k0);
    MtStage<BN, B_ACROSS> sb(b, n0, k0);
#pragma unroll
    for (int m = 0; m < S::MA; ++m)
#pragma unroll
        for (int n = 0; n < S::NB; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.f;
    if (nk <= 0) return;
    sa.issue(lds);
    sb.issue(lds + A_BYTES);
    __syncthreads();  // waits for the copies as well
    for (int kt = 0; kt < nk; ++kt) {
        unsigned char* cur = lds + (kt & 1) * BUF;
        if (kt + 1 < nk) {
            unsigned char* nxt = lds + ((kt + 1) & 1) * BUF;
            sa.issue(nxt);
            sb.issue(nxt + A_BYTES);
        }
        // Four sub-steps of 16 k with two register sets of fragments: the reads of sub-step s + 1 go out between the
        // products of sub-step s, so the matrix pipe waits for LDS once per step of 64.
        auto read_set = [&](int sub, mt_s16x8* fa, mt_s16x8* fb) {
#pragma unroll
            for (int m = 0; m < S::MA; ++m) fa[m] = mt_fragment<MT_BM, A_ACROSS>(cur, wm * S::MA * 32 + m * 32, sub);
#pragma unroll
            for (int n = 0; n < S::NB; ++n) fb[n] = mt_fragment<BN, B_ACROSS>(cur + A_BYTES, wn * S::NB * 32 + n * 32, sub);
        };
        auto multiply = [&](const mt_s16x8* fa, const mt_s16x8* fb) {
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int n = 0; n < S::NB; ++n)
                    acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[m], fb[n], acc[m][n], 0, 0, 0);
        };
        mt_s16x8 fa0[S::MA], fb0[S::NB], fa1[S::MA], fb1[S::NB];
        constexpr int READS = S::MA * (A_ACROSS ? 2 : 1) + S::NB * (B_ACROSS ? 2 : 1), PRODUCTS = S::MA * S::NB;
        constexpr int PER = (READS + PRODUCTS - 1) / PRODUCTS;
        auto interleave = [&]() {
#pragma unroll
            for (int i = 0; i < PRODUCTS; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
            }
        };
        read_set(0, fa0, fb0);
        __builtin_amdgcn_sched_barrier(0);
        read_set(1, fa1, fb1);
        multiply(fa0, fb0);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
        read_set(2, fa0, fb0);
        multiply(fa1, fb1);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
        read_set(3, fa1, fb1);
        multiply(fa0, fb0);
        interleave();
        __builtin_amdgcn_sched_barrier(0);
        multiply(fa1, fb1);
        __syncthreads();  // the next tiles have landed, and everybody is done with these
    }
}

// Workgroups are dealt to the eight XCDs round robin; every XCD takes one contiguous stretch of the tiles, ordered
// in groups of eight n tiles that walk the m tiles together: the 32 workgroups an XCD runs at a time share about
// four m tiles and eight n tiles in its L2.
__device__ __forceinline__ void mt_tile(int block, int m_tiles, int n_tiles, int& tm, int& tn) {
    const int total = m_tiles * n_tiles;
    const int xcd = block & 7, slot = block >> 3;
    const int per = total >> 3, extra = total & 7;
    const int id = xcd * per + (xcd < extra ? xcd : extra) + slot;
    const int group = id / (8 * m_tiles);
    const int in_group = n_tiles - group * 8 < 8 ? n_tiles - group * 8 : 8;
    const int rest = id - group * 8 * m_tiles;
    tm = rest / in_group;
    tn = group * 8 + rest - tm * in_group;
}
