// Log-probabilities and entropies of tokens from hidden states [N, H] and the output projection [V, H]: what
// token_logps.hip computes from logits.  Forward, the products of a 256 x BN tile are consumed where they are: a row
// keeps (max, sum of exponentials, weighted sum) per 256 columns and its own token's logit.  Backward, the products --
// kept in fp32 if the caller gave room, or formed again -- are turned into the logits' gradient G = dL/dlogits in chunks of
// columns, and
//   d hidden = G x weight (sum over v),    d weight = G^T x hidden (sum over rows)
// follow with fp32 accumulators.  The matrix cores take G in bf16 or not at all, and bf16 alone is not enough: rounded to it
// once, elements that cancel (rows that share a hidden state and whose gradients add up to 0, as a group's do at its first
// token) leave 2^-8 of what they were.  So G is held in two bf16 pieces, its rounding and what that leaves: off by at most
// 2^-16 of each element, and each of its two products is made twice, with the same accumulators.  Five or six products of
// 2 N V H where three (or four, formed again) would do in bf16: 8192 rows of H = 2048, V = 152,640 with both gradients 21.1 ms,
// 13.7 with G in bf16.  Bound by the matrix cores at many rows, by the weight (V H elements read per product, written
// once) at few.
#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "common.h"
#include "lse_math.h"
#include "mfma_tile.h"

#define LL_FLOOR (-200.f)           // 2^-200 is 0 in fp32: keeps 0 * -inf out of the entropy sums
#define LL_CUS 256
#define LL_CHUNK_BYTES (1ll << 30)  // G of one chunk, both pieces

// The rows that count are brought together first: what follows works on `plan[0]` rows, a number that only the device
// knows, and padding costs nothing but its place in the scratch memory (1403 rows, H = 3584, V = 151,669, with the gradient
// of hidden, nothing kept: half of them padding 2.7 ms, none 5.1; bringing 320 rows together takes 15 us of 1320).
struct LlOperands {
    const uint16_t* weight;     // [V, H]
    int64_t weight_ld;
    const uint16_t* hidden;     // [rows, H], the rows that count
    const int* plan;            // LL_PLAN_*
    int H, V;
};
#define LL_PLAN_ROWS 0          // rows that count
#define LL_PLAN_SPLITS 1        // splits of d hidden's sum

struct LlCompact {
    const uint16_t* hidden;     // [N, H]
    int64_t hidden_ld;
    const int64_t* ids;         // [N]
    int N, H, V;
    const int* offsets;         // [ceil(N / 16)] rows that count in front of every 16; null: each workgroup counts them
    uint16_t* to;               // [rows, H]
    int* plan;
    int* tok;                   // [rows] the row's token
    // forward: row_of [rows], and the results of the rows that do not count
    int* row_of;
    float* logps;
    float2* stats;
    float* entropy;
    // backward
    const float* g;
    const float* h;
    float inv_t;
    int* pos;                   // [N] place among the rows that count, or -1
    struct LlRow* rows;
    int dh_bn, h_tiles, steps, slab_rows;  // what splits are chosen by
    bool kept;                  // rows are as in the forward pass: those whose gradients are 0 keep their places
};

// What a row needs to turn a product into its gradient: w = 2^((x - m) k), G = w (alpha + beta (x - m) k) + at at the
// token; tok = -1: nothing flows into this row, its G is 0 whatever the products are.
struct LlRow {
    float m, alpha, beta, at;
    int tok;
    int pad[3];
};

// Splits of d hidden's sum: as many as fill the CUs evenly, each at least eight steps long.
__host__ __device__ static int ll_splits(int rows, int bn, int h_tiles, int steps, int slab_rows) {
    const int64_t tiles = (int64_t)((rows + bn - 1) / bn) * h_tiles;
    if (tiles >= 16 * LL_CUS || rows <= 0) return 1;
    const int by_steps = steps / 8, by_room = slab_rows / rows, both = by_steps < by_room ? by_steps : by_room;
    const int most = both < 64 ? both : 64;
    int best = 1;
    float best_use = 0.f;
    for (int s = 1; s == 1 || s <= most; ++s) {
        const int wgs = (int)tiles * s;
        const float use = (float)wgs / (float)((wgs + LL_CUS - 1) / LL_CUS * LL_CUS);
        if (use > best_use + 0.04f) {
            best_use = use;
            best = s;
        }
    }
    return best;
}

// Backward, rows whose gradients are 0 do not count either (but for their places, with kept logits).
__device__ __forceinline__ bool ll_live(const LlCompact& a, int r) { return (a.g && a.g[r] != 0.f) || (a.h && a.h[r] != 0.f); }
template <bool BACK>
__device__ __forceinline__ bool ll_counts(const LlCompact& a, int r) {
    return r < a.N && a.ids[r] >= 0 && (!BACK || a.kept || ll_live(a, r));
}

template <bool BACK>
__global__ __launch_bounds__(1024) void lm_logps_offsets_kernel(LlCompact a, int* offsets, int n) {
    __shared__ int part[16];
    int all = 0;
    for (int base = 0; base < n; base += 1024) {
        const int i = base + threadIdx.x;
        int mine = 0;
        if (i < n)
            for (int j = 0; j < 16; ++j) mine += ll_counts<BACK>(a, i * 16 + j) ? 1 : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(upto, o, 64);
            if ((threadIdx.x & 63) >= o) upto += x;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = upto;
        __syncthreads();
        int before = all + upto - mine;
        for (int w = 0; w < 16; ++w) {
            if (w < (int)(threadIdx.x >> 6)) before += part[w];
            all += part[w];
        }
        if (i < n) offsets[i] = before;
    }
}

// Workgroup (16 rows, 512 h).
template <bool BACK>
__global__ __launch_bounds__(256) void lm_logps_compact_kernel(LlCompact a) {
    __shared__ int part[4], place[16];
    const int r0 = blockIdx.x * 16;
    int before = 0;
    if (a.offsets == nullptr) {
#pragma unroll 4
        for (int i = threadIdx.x; i < r0; i += 256) before += ll_counts<BACK>(a, i) ? 1 : 0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, 64);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = before;
        __syncthreads();
        before = part[0] + part[1] + part[2] + part[3];
    } else {
        before = a.offsets[blockIdx.x];
    }
    if (threadIdx.x < 64) {
        const bool counts = threadIdx.x < 16 && ll_counts<BACK>(a, r0 + threadIdx.x);
        const uint64_t mask = __ballot(counts);
        const int at = before + __popcll(mask & ((1ull << threadIdx.x) - 1));
        if (threadIdx.x < 16) place[threadIdx.x] = counts ? at : -1;
        const int r = r0 + threadIdx.x;
        if (blockIdx.y == 0 && threadIdx.x < 16 && r < a.N) {
            if constexpr (BACK) {
                const bool live = counts && ll_live(a, r);
                a.pos[r] = live ? at : -1;
                if (counts && !live) {
                    a.rows[at] = {0.f, 0.f, 0.f, 0.f, -1, {0, 0, 0}};
                    a.tok[at] = -1;
                }
                if (live) {
                    const int64_t id = a.ids[r];
                    const float g = a.g ? a.g[r] : 0.f, h = a.h ? a.h[r] : 0.f;
                    const float2 st = a.stats[r];
                    const float ln2 = 0.69314718055994531f;
                    LlRow o = {st.x, 0.f, 0.f, 0.f, 0, {0, 0, 0}};
                    o.alpha = -(g + (a.h ? h * (a.entropy[r] - log2f(st.y) * ln2) : 0.f)) * a.inv_t / st.y;
                    o.beta = -h * ln2 * a.inv_t / st.y;
                    o.at = g * a.inv_t;
                    if (id >= a.V) o.alpha = NAN;
                    o.tok = id < a.V ? (int)id : 0;
                    a.rows[at] = o;
                    a.tok[at] = o.tok;
                }
            } else if (counts) {
                const int64_t id = a.ids[r];
                a.row_of[at] = r;
                a.tok[at] = id < a.V ? (int)id : a.V;
            } else {
                a.logps[r] = 0.f;
                a.stats[r] = make_float2(0.f, 1.f);
                if (a.entropy) a.entropy[r] = 0.f;
            }
        }
        if (r0 + 16 >= a.N && blockIdx.y == 0 && threadIdx.x == 0) {  // the last 16
            const int rows = before + __popcll(mask);
            a.plan[LL_PLAN_ROWS] = rows;
            if (BACK) a.plan[LL_PLAN_SPLITS] = ll_splits(rows, a.dh_bn, a.h_tiles, a.steps, a.slab_rows);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 4 + (threadIdx.x >> 6), at = place[row], h = blockIdx.y * 512 + (threadIdx.x & 63) * 8;
        if (at >= 0 && h < a.H)
            *reinterpret_cast<u32x4*>(a.to + (int64_t)at * a.H + h) =
                *reinterpret_cast<const u32x4*>(a.hidden + (int64_t)(r0 + row) * a.hidden_ld + h);
    }
}

struct LlArgs {
    LlOperands o;
    int m_tiles;
    float k;                    // log2(e) / temperature
    const int* tok;             // [rows]
    float2* partials;           // [parts][n_pad] (max, sum), parts = m_tiles x waves along m
    float* weighted;            // [parts][n_pad], with entropies
    int64_t n_pad;
    float* chosen;              // [rows] logit of the row's token
    float* kept;                // null, or all products as they lie in the registers: [V / 32][n_pad / 32][4][64 lanes][4]
};

template <int BN>
using LlLogits = MtPipe<BN, MtAlong<MT_BM, BN>, MtReadAlong, MtAlong<BN, BN>, MtReadAlong>;

template <int BN>
__device__ __forceinline__ void ll_begin(LlLogits<BN>& pipe, const LlOperands& o, int rows, int v0, int r0) {
    pipe.begin(MtAlong<MT_BM, BN>(o.weight, o.weight_ld, o.V, v0, 0), MtAlong<BN, BN>(o.hidden, o.H, rows, r0, 0), o.H / MT_BK);
}

// Element `at` of a lane's row n: selected, where branches would make a jump table of stores.
template <int MA, int NB>
__device__ __forceinline__ float ll_pick(const mt_f32x16 (&acc)[MA][NB], int n, int at) {
    float v = acc[0][n][0];
#pragma unroll
    for (int m = 0; m < MA; ++m)
#pragma unroll
        for (int e = 0; e < 16; ++e) v = m * 16 + e == at ? acc[m][n][e] : v;
    return v;
}

// As many workgroups as run at a time; each takes every gridDim-th tile and starts the next one's copies before it
// turns to its own results.  Those stay inside the wave: a row's sums over the wave's columns are one partial.
// H = 2048, V = 152,640: 8192 rows 3.70 ms (1.38 PFLOP/s; the library's product of these operands alone 3.72 ms), 320
// rows 227 us, 64 rows and fewer 147 us (4.3 TB/s of weight: rows are fetched 128 bytes at a time).
template <int BN, bool ENT, bool KEEP>
__device__ __forceinline__ void ll_forward_tiles(const LlArgs& a) {
    typedef MtShape<BN> S;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = mt_wave();
    const int wm = wave / S::WN, wn = wave % S::WN, half = lane >> 5;
    const int rows = a.o.plan[LL_PLAN_ROWS], n_tiles = (rows + BN - 1) / BN, tiles = a.m_tiles * n_tiles;
    if ((int)blockIdx.x >= tiles) return;
    LlLogits<BN> pipe(lds);
    int tm, tn;
    mt_tile(blockIdx.x, a.m_tiles, n_tiles, tm, tn);
    ll_begin(pipe, a.o, rows, tm * MT_BM, tn * BN);
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int v0 = tm * MT_BM, r0 = tn * BN, part = tm * S::WM + wm;
        int id[S::NB];
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int r = r0 + (wn * S::NB + n) * 32 + (lane & 31);
            id[n] = r < rows ? a.tok[r] : -1;
        }
        typename LlLogits<BN>::Acc acc;
        pipe.clear(acc);
        // the stores of the tile before's sums, and products
        pipe.template run<S::NB + (KEEP ? S::MA * S::NB * 4 : 0)>(acc, tile != (int)blockIdx.x);
#pragma unroll
        for (int n = 0; n < S::NB; ++n) asm volatile("" : "+v"(id[n]));  // waited for here, not behind the next copies
        if (tile + (int)gridDim.x < tiles) {
            mt_tile(tile + gridDim.x, a.m_tiles, n_tiles, tm, tn);
            ll_begin(pipe, a.o, rows, tm * MT_BM, tn * BN);
        }
        const int vw = v0 + wm * S::MA * 32 + 4 * half;  // vocabulary entry of m = 0, e = 0
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int r = r0 + (wn * S::NB + n) * 32 + (lane & 31);
            if constexpr (KEEP) {
                const int n32 = r0 / 32 + wn * S::NB + n;
#pragma unroll
                for (int m = 0; m < S::MA; ++m) {
                    float* const to = a.kept + ((int64_t)((v0 >> 5) + wm * S::MA + m) * (a.n_pad >> 5) + n32) * 1024 + lane * 4;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<mt_f32x4*>(to + q * 256) =
                            mt_f32x4{acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]};
                }
            }
            if (v0 + MT_BM > a.o.V) {  // the last tile
#pragma unroll
                for (int m = 0; m < S::MA; ++m)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (vw + m * 32 + (e & 3) + 8 * (e >> 2) >= a.o.V) acc[m][n][e] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[m][n][e]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));  // the other half of the lanes holds the same row
            const float ref = mx == -INFINITY ? 0.f : mx;
            float s0 = 0.f, s1 = 0.f, u = 0.f;
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float t = (acc[m][n][e] - ref) * a.k;
                    const float w = fast_exp2(t);
                    if (e & 1) s1 += w; else s0 += w;
                    if (ENT) u = fmaf(w, fmaxf(t, LL_FLOOR), u);
                }
            float s = s0 + s1;
            s += __shfl_xor(s, 32, 64);
            if (ENT) u += __shfl_xor(u, 32, 64);
            if (half == 0) {
                a.partials[(int64_t)part * a.n_pad + r] = make_float2(mx, s);
                if (ENT) a.weighted[(int64_t)part * a.n_pad + r] = u;
            }
            const int off = id[n] - vw;  // runs of four entries, every eight
            if (id[n] >= vw && id[n] < vw + S::MA * 32 && (off & 4) == 0) {
                const int at = (off >> 5) * 16 + ((off & 31) >> 3) * 4 + (off & 3);
                a.chosen[r] = ll_pick<S::MA, S::NB>(acc, n, at);
            }
        }
    }
}

template <int BN, bool ENT>
__global__ __launch_bounds__(MtShape<BN>::THREADS) void lm_logps_kernel(LlArgs a) {
    ll_forward_tiles<BN, ENT, false>(a);
}

template <int BN, bool ENT>
__global__ __launch_bounds__(MtShape<BN>::THREADS) void lm_logps_keep_kernel(LlArgs a) {
    ll_forward_tiles<BN, ENT, true>(a);
}

struct LlJoin {
    LlArgs g;
    int parts;
    float* logps;
    float2* stats;
    float* entropy;
    const int* row_of;         // [rows]
};

// Joins a row's partials, ROWS rows per workgroup.
template <int ROWS>
__global__ __launch_bounds__(256) void lm_logps_join_kernel(LlJoin a) {
    constexpr int PER = 256 / ROWS;  // threads a row
    __shared__ float sm[PER][ROWS + 1], ss[PER][ROWS + 1], su[PER][ROWS + 1];
    const int i = threadIdx.x % ROWS, j = threadIdx.x / ROWS;
    const int r = blockIdx.x * ROWS + i, rows = a.g.o.plan[LL_PLAN_ROWS];
    if ((int)blockIdx.x * ROWS >= rows) return;  // rows of the last 16 past the end read what a clamped row left
    const float k = a.g.k;
    float m = -INFINITY, s = 0.f, u = 0.f;
    auto add = [&](float pm, float ps, float pu) {
        const float mn = fmaxf(m, pm);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float da = fmaxf((m - ref) * k, LL_FLOOR), db = fmaxf((pm - ref) * k, LL_FLOOR);
        const float fa = fast_exp2(da), fb = fast_exp2(db);
        u = (u + s * da) * fa + (pu + ps * db) * fb;
        s = s * fa + ps * fb;
        m = mn;
    };
    for (int t = j; t < a.parts; t += PER) {
        const float2 p = a.g.partials[(int64_t)t * a.g.n_pad + r];
        add(p.x, p.y, a.entropy ? a.g.weighted[(int64_t)t * a.g.n_pad + r] : 0.f);
    }
    sm[j][i] = m;
    ss[j][i] = s;
    su[j][i] = u;
#pragma unroll
    for (int half = PER / 2; half > 0; half >>= 1) {  // in a fixed order
        __syncthreads();
        if (j < half) {
            add(sm[j + half][i], ss[j + half][i], su[j + half][i]);
            sm[j][i] = m;
            ss[j][i] = s;
            su[j][i] = u;
        }
    }
    if (j != 0 || r >= rows) return;
    const int id = a.g.tok[r], row = a.row_of[r];
    const float ln2 = 0.69314718055994531f;
    const float ls = log2f(s);
    a.logps[row] = id < a.g.o.V ? ((a.g.chosen[r] - m) * k - ls) * ln2 : NAN;
    a.stats[row] = make_float2(m, s);
    if (a.entropy) a.entropy[row] = (ls - u / s) * ln2;
}

// ---- backward -----------------------------------------------------------------------------------------
// Hidden in fragment blocks of 32 h x 16 n, [64 n][H / 32][4], for d weight: workgroup (64 rows, 32 h).  Rows past the
// end, and rows without a gradient, are 0.
__global__ __launch_bounds__(256) void lm_logps_prepare_kernel(LlOperands o, const int* tok, char* copy) {
    const int r0 = blockIdx.x * 64, rows = o.plan[LL_PLAN_ROWS];
    if (r0 >= rows) return;
    const int lane = threadIdx.x & 63, n0 = r0 + (threadIdx.x >> 6) * 16 + (lane >> 5) * 8, h = blockIdx.y * 32 + (lane & 31);
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
    u16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = n0 + j < rows && tok[n0 + j] >= 0 ? o.hidden[(int64_t)(n0 + j) * o.H + h] : (uint16_t)0;
    *reinterpret_cast<u16x8*>(copy + ((int64_t)blockIdx.x * (o.H / 32) + blockIdx.y) * 4096 + threadIdx.x * 16) = v;
}

// G of a chunk of columns, in fragment blocks of 32 n x 16 v, [64 n][2 pieces][64 v][2][4]: a wave's results are such
// blocks already, so a store is 1 KB at a time, and both products read it 8 KB and more at a time.  8192 rows as
// above: 4.30 ms (1.19 PFLOP/s; one piece 3.80).
struct LlGrad {
    LlOperands o;
    int m_tiles;
    int v_begin, v64;          // first column of the chunk, its width in 64s
    float k;
    const LlRow* rows;
    char* out;
};

template <int BN, bool ENT>
__global__ __launch_bounds__(MtShape<BN>::THREADS) void lm_logps_dlogits_kernel(LlGrad a) {
    typedef MtShape<BN> S;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = mt_wave();
    const int wm = wave / S::WN, wn = wave % S::WN, half = lane >> 5;
    const int rows = a.o.plan[LL_PLAN_ROWS], n_pad = (rows + 63) / 64 * 64;  // rows of G
    const int n_tiles = (rows + BN - 1) / BN, tiles = a.m_tiles * n_tiles;
    const int64_t piece = (int64_t)a.v64 * 8192;  // from the first to the second
    if ((int)blockIdx.x >= tiles) return;
    LlLogits<BN> pipe(lds);
    int tm, tn;
    mt_tile(blockIdx.x, a.m_tiles, n_tiles, tm, tn);
    ll_begin(pipe, a.o, rows, a.v_begin + tm * MT_BM, tn * BN);
    constexpr int STORES = S::MA * S::NB * 4;
    bool stored = false;  // all STORES of the tile before were made
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int v0 = a.v_begin + tm * MT_BM, r0 = tn * BN;
        LlRow row[S::NB];
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int r = r0 + (wn * S::NB + n) * 32 + (lane & 31);
            row[n] = a.rows[r < rows ? r : rows - 1];
            if (r >= rows) row[n].tok = -1;  // G is 0 whatever the products are
        }
        const int v64 = tm * 4;
        typename LlLogits<BN>::Acc acc;
        pipe.clear(acc);
        pipe.template run<STORES>(acc, stored);
#pragma unroll
        for (int n = 0; n < S::NB; ++n)  // waited for here, not behind the next copies
            asm volatile("" : "+v"(row[n].m), "+v"(row[n].alpha), "+v"(row[n].beta), "+v"(row[n].at), "+v"(row[n].tok));
        stored = r0 + (wn + 1) * S::NB * 32 <= n_pad;
        if (tile + (int)gridDim.x < tiles) {
            mt_tile(tile + gridDim.x, a.m_tiles, n_tiles, tm, tn);
            ll_begin(pipe, a.o, rows, a.v_begin + tm * MT_BM, tn * BN);
        }
        const int vw = v0 + wm * S::MA * 32 + 4 * half;
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int n32 = r0 / 32 + wn * S::NB + n;
            if (n32 * 32 >= n_pad) continue;
            char* const out = a.out + ((int64_t)(n32 >> 1) * 2 * a.v64 + v64) * 8192 + (n32 & 1) * 4096 + lane * 16;
            const float m0 = row[n].m, alpha = row[n].alpha, beta = row[n].beta;
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float t = (acc[m][n][e] - m0) * a.k;
                    acc[m][n][e] = fast_exp2(t) * (ENT ? fmaf(beta, fmaxf(t, LL_FLOOR), alpha) : alpha);
                }
            const int off = row[n].tok - vw;  // runs of four entries, every eight
            if (row[n].tok >= 0 && off >= 0 && off < S::MA * 32 && (off & 4) == 0) {
                const int at = (off >> 5) * 16 + ((off & 31) >> 3) * 4 + (off & 3);
#pragma unroll
                for (int m = 0; m < S::MA; ++m)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[m][n][e] += m * 16 + e == at ? row[n].at : 0.f;
            }
            const bool dead = row[n].tok < 0;
            if (__any(dead)) {
#pragma unroll
                for (int m = 0; m < S::MA; ++m)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[m][n][e] = dead ? 0.f : acc[m][n][e];
            }
            if (v0 + MT_BM > a.o.V) {  // the last tile
#pragma unroll
                for (int m = 0; m < S::MA; ++m)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (vw + m * 32 + (e & 3) + 8 * (e >> 2) >= a.o.V) acc[m][n][e] = 0.f;
            }
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const mt_f32x16& c = acc[m][n];
                    const mt_f32x4 x = {c[8 * q], c[8 * q + 1], c[8 * q + 2], c[8 * q + 3]};
                    const mt_f32x4 y = {c[8 * q + 4], c[8 * q + 5], c[8 * q + 6], c[8 * q + 7]};
                    const int v16 = (wm * S::MA + m) * 2 + q;
                    char* const to = out + (v16 >> 2) * 8192 + (v16 & 3) * 1024;
                    *reinterpret_cast<mt_u32x4*>(to) = mt_pack8(x, y);
                    *reinterpret_cast<mt_u32x4*>(to + piece) = mt_pack8(mt_rest(x), mt_rest(y));
                }
        }
    }
}

// G from the products that the forward pass kept, a wave a block of 32 v x 32 n: bound by HBM.  8192 rows as above: 1.62
// ms (10 GB, 6.2 TB/s) instead of 4.30; keeping them adds 0.4 ms to the forward pass.  320 rows: 61 us instead of 255, 44
// more forward.
template <bool ENT>
__global__ __launch_bounds__(256) void lm_logps_kept_kernel(LlGrad a, const float* kept, int n32s) {
    const int lane = threadIdx.x & 63, wave = mt_wave(), half = lane >> 5;
    const int n32 = blockIdx.y, rows = a.o.plan[LL_PLAN_ROWS], r = n32 * 32 + (lane & 31);
    if ((n32 & ~1) * 32 >= rows) return;  // G has whole pairs of blocks
    LlRow row = a.rows[r < rows ? r : rows - 1];
    if (r >= rows) row.tok = -1;
    const int v32 = blockIdx.x * 4 + wave;  // of the chunk
    if (v32 >= a.m_tiles * 8) return;
    const int vw = a.v_begin + v32 * 32 + 4 * half;
    float x[16];
    const float* const from = kept + ((int64_t)((a.v_begin >> 5) + v32) * n32s + n32) * 1024 + lane * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const mt_f32x4 v = __builtin_nontemporal_load(reinterpret_cast<const mt_f32x4*>(from + q * 256));
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * q + j] = v[j];
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float t = (x[e] - row.m) * a.k;
        x[e] = fast_exp2(t) * (ENT ? fmaf(row.beta, fmaxf(t, LL_FLOOR), row.alpha) : row.alpha);
    }
    const int off = row.tok - vw;  // runs of four entries, every eight
    if (row.tok >= 0 && off >= 0 && off < 32 && (off & 4) == 0) {
        const int at = (off >> 3) * 4 + (off & 3);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] += e == at ? row.at : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
        if (row.tok < 0 || vw + (e & 3) + 8 * (e >> 2) >= a.o.V) x[e] = 0.f;
    const int64_t piece = (int64_t)a.v64 * 8192;  // from the first to the second
    char* const out = a.out + ((int64_t)(n32 >> 1) * 2 * a.v64 + (v32 >> 1)) * 8192 + (n32 & 1) * 4096 + (v32 & 1) * 2048 + lane * 16;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const mt_f32x4 lo = {x[8 * q], x[8 * q + 1], x[8 * q + 2], x[8 * q + 3]};
        const mt_f32x4 hi = {x[8 * q + 4], x[8 * q + 5], x[8 * q + 6], x[8 * q + 7]};
        *reinterpret_cast<mt_u32x4*>(out + q * 1024) = mt_pack8(lo, hi);
        *reinterpret_cast<mt_u32x4*>(out + piece + q * 1024) = mt_pack8(mt_rest(lo), mt_rest(hi));
    }
}

// d hidden: C[n][h] = sum over the chunk's columns of G[n][v] weight[v][h], fp32 slabs, one per split of the columns.
// Both pieces of G: 8192 rows 7.67 ms (1.34 PFLOP/s; the library's product with one 3.62 ms).
struct LlDh {
    LlOperands o;
    const char* g;
    int m_tiles, steps, v_begin, v64;
    int add;                   // 1: go on from what the chunk before left
    float* slabs;              // [splits][rows][H]
};

template <int BN>
__global__ __launch_bounds__(MtShape<BN>::THREADS) void lm_logps_dhidden_kernel(LlDh a) {
    typedef MtShape<BN> S;
    extern __shared__ __align__(16) unsigned char lds[];
    const int rows = a.o.plan[LL_PLAN_ROWS], splits = a.o.plan[LL_PLAN_SPLITS], n_tiles = (rows + BN - 1) / BN;
    const int total = splits * a.m_tiles * n_tiles, steps_per = (a.steps + splits - 1) / splits;
    const int lane = threadIdx.x & 63, wave = mt_wave();
    const int wm = wave / S::WN, wn = wave % S::WN, half = lane >> 5;
    const int64_t piece = (int64_t)a.v64 * 8192;
    MtPipe<BN, MtAcross<BN>, MtReadAcross, MtBlocksAlong<BN, BN>, MtReadBlocksAlong> pipe(lds);
    for (int block = blockIdx.x; block < total; block += gridDim.x) {
        // one XCD takes neighbouring tiles: all h tiles of a few n tiles, which share G
        const int xcd = block & 7;
        const int id = xcd * (total >> 3) + (xcd < (total & 7) ? xcd : total & 7) + (block >> 3);
        const int tm = id % a.m_tiles, rest = id / a.m_tiles;
        const int tn = rest % n_tiles, split = rest / n_tiles;
        const int h0 = tm * MT_BM, r0 = tn * BN;
        const int s0 = split * steps_per, s1 = s0 + steps_per < a.steps ? s0 + steps_per : a.steps;
        typename decltype(pipe)::Acc acc;
        pipe.begin(MtAcross<BN>(a.o.weight + (int64_t)a.v_begin * a.o.weight_ld, a.o.weight_ld, a.o.H, a.o.V - a.v_begin, h0, s0 * MT_BK),
                   MtBlocksAlong<BN, BN>(a.g + ((int64_t)(r0 / 64) * 2 * a.v64 + s0) * 8192, piece, 8192 - piece,
                                         (uint32_t)a.v64 * 16384u, (rows + 63) / 64 * 2 - r0 / 32),
                   (s1 - s0) * 2);
        float* slab = a.slabs + (int64_t)split * rows * a.o.H;
        pipe.clear(acc);
        if (a.add) {
#pragma unroll
            for (int n = 0; n < S::NB; ++n) {
                const int r = r0 + (wn * S::NB + n) * 32 + (lane & 31);
                if (r >= rows) continue;
#pragma unroll
                for (int m = 0; m < S::MA; ++m) {
                    const int h = h0 + (wm * S::MA + m) * 32;
                    if (h < a.o.H) pipe.load(acc, m, n, slab + (int64_t)r * a.o.H + h);
                }
            }
        }
        pipe.run(acc);
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int r = r0 + (wn * S::NB + n) * 32 + (lane & 31);
            if (r >= rows) continue;
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int h = h0 + (wm * S::MA + m) * 32 + 8 * q + 4 * half;
                    if (h >= a.o.H) continue;
                    mt_f32x4* o = reinterpret_cast<mt_f32x4*>(slab + (int64_t)r * a.o.H + h);
                    *o = mt_f32x4{acc[m][n][q * 4], acc[m][n][q * 4 + 1], acc[m][n][q * 4 + 2], acc[m][n][q * 4 + 3]};
                }
        }
    }
}

// Sum of the slabs in their order, rounded once.
__global__ __launch_bounds__(256) void lm_logps_dhidden_join_kernel(LlOperands o, int N, const float* slabs, const int* pos,
                                                                    uint16_t* out) {
    const int64_t n = (int64_t)N * o.H, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    const int row = (int)(i / o.H), h = (int)(i - (int64_t)row * o.H), r = pos[row];
    mt_f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (r >= 0) {
        const int splits = o.plan[LL_PLAN_SPLITS];
        const int64_t slab = (int64_t)o.plan[LL_PLAN_ROWS] * o.H, at = (int64_t)r * o.H + h;
        for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const mt_f32x4*>(slabs + s * slab + at);
    }
    *reinterpret_cast<mt_b16x4*>(out + i) = __builtin_convertvector(v, mt_b16x4);
}

// d weight of the chunk: C[v][h] = sum over the rows of G[n][v] hidden[n][h], both pieces of G.  8192 rows: 7.7 ms (1.33
// PFLOP/s; the library's product with one 4.40 ms).  At few rows the stores come on top of the products (a wave's copies are
// counted together with its stores, so the copies of a tile's third step wait for the stores of the tile before): 320 rows 430 us.
struct LlDw {
    const char* copy;
    const char* g;
    int H, V;
    int m_tiles, n_tiles, v_begin, v64;
    const int* plan;
    uint16_t* out;             // [V][H]
};

// LINES: two buffers of either operand, and the LDS left holds the results on their way to whole lines of 128 bytes;
// otherwise three buffers of G and stores of the 16 bytes that a lane holds.  Up to LL_LINES_STEPS steps (two for every 64
// rows) the stores weigh more: the backward pass for d weight alone takes, with lines and without, at H = 2048 and V = 152,640
// (625 MB to write) 64 rows 158 and 244 us, 320 rows 427 and 530, 512 rows 710 and 731, 768 rows 1011 and 997, 1024 rows 1310
// and 1277; at H = 3584 and V = 40,000 64 rows 84 and 101, 512 rows 296 and 323, 1024 rows 525 and 552.
#define LL_LINES_STEPS 16
template <bool LINES>
using LlDwPipe = MtPipe<256, MtBlocksAlong<MT_BM, 256>, MtReadBlocksAlong, MtBlocksAcross, MtReadBlocksAcross, !LINES, LINES ? 2 : 3>;

// Eight v tiles at a time, one per XCD, all h tiles of each: G is read by one XCD.
__device__ __forceinline__ void ll_dw_at(const LlDw& a, int tile, int& h0, int& c0) {
    const int group = tile / (8 * a.m_tiles), left = a.n_tiles - group * 8, wide = left < 1 ? 1 : left < 8 ? left : 8;
    const int rest = tile - group * 8 * a.m_tiles;
    h0 = rest / wide * MT_BM;
    c0 = (group * 8 + rest % wide) * 256;
}

template <bool LINES>
__device__ __forceinline__ void ll_dw_begin(LlDwPipe<LINES>& pipe, const LlDw& a, int rows, int tile, int& h0, int& c0) {
    ll_dw_at(a, tile, h0, c0);
    pipe.begin(MtBlocksAlong<MT_BM, 256>(a.copy + (int64_t)(h0 / 32) * 4096, 0, (int64_t)(a.H / 32) * 4096, 8192u, a.H / 32 - h0 / 32),
               MtBlocksAcross(a.g + (int64_t)(c0 / 64) * 8192, (int64_t)a.v64 * 8192), (rows + MT_BK - 1) / MT_BK * 2);
}

template <bool LINES>
__global__ __launch_bounds__(MtShape<256>::THREADS) void lm_logps_dweight_kernel(LlDw a) {
    typedef MtShape<256> S;
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = mt_wave();
    const int wm = wave / S::WN, wn = wave % S::WN;
    const int tiles = a.m_tiles * a.n_tiles, rows = a.plan[LL_PLAN_ROWS];
    LlDwPipe<LINES> pipe(lds);
    // LINES: behind the 128 KB of the pipe, 4 KB of each wave
    const uint32_t staging = (uint32_t)(uintptr_t)(mt_lds_void*)lds + 4 * MT_BM * MT_BK * 2 + wave * 4096;
    int h_next, c_next;
    ll_dw_begin<LINES>(pipe, a, rows, blockIdx.x, h_next, c_next);
    constexpr int STORES = S::MA * S::NB * 2;
    bool stored = false;  // all STORES of the tile before were made
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int h0 = h_next, c0 = c_next;
        typename LlDwPipe<LINES>::Acc acc;
        pipe.clear(acc);
        pipe.template run<STORES>(acc, stored);
        stored = a.v_begin + c0 + (wn + 1) * S::NB * 32 <= a.V && h0 + (wm + 1) * S::MA * 32 <= a.H;
        if (tile + (int)gridDim.x < tiles) ll_dw_begin<LINES>(pipe, a, rows, tile + gridDim.x, h_next, c_next);
#pragma unroll
        for (int n = 0; n < S::NB; ++n) {
            const int v = a.v_begin + c0 + (wn * S::NB + n) * 32;
            uint16_t* const out = a.out + (int64_t)v * a.H;
#pragma unroll
            for (int m = 0; m < S::MA; m += 2) {
                const int h = h0 + (wm * S::MA + m) * 32;
                if (h >= a.H) continue;
                if constexpr (LINES) mt_store_rows(acc[m][n], acc[m + 1][n], staging, out + h, a.H, a.V - v);
                else if (v + (lane & 31) < a.V) mt_store_lanes(acc[m][n], acc[m + 1][n], out + (int64_t)(lane & 31) * a.H + h);
            }
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------
static int64_t ll_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Rows per tile of the products with the logits' shape (m_tiles x n tiles of 256 x BN): what counts is whole rounds over
// the CUs.  At H = 2048 a round takes 54 us with tiles of 256 rows, 45 with 192, 34 with 128, 41 with 64 (two to a CU).
// At V = 152,640 320 rows take 230 us in 5 rounds of 192, 237 in 7 of 128 and 270 in 5 of 256; 576 rows 310, 374 and 380;
// 400 rows 270 in 5 rounds of 256 and 309 in 10 of 128.  Whole calls from 32 to 1403 rows at H = 576, 1536, 2048 and 3584: what is chosen
// is at most 8 % behind the best of the four (H = 3584: 320 rows 379 us, 476, 403, 380 and 437 with 64, 128, 192 and 256; 64 rows
// 236 with 64, 223 with 128); at V = 40,000 at most 18 % (H = 2048, 150 and 192 rows: 51 us with 64 and 44 with 192).
static double ll_cost(int bn) { return bn == 64 ? 0.4 : bn == 128 ? 0.64 : bn == 192 ? 0.84 : 1.0; }

static int ll_bn(int N, int64_t m_tiles) {
    int best = 0;
    double least = 0.0;
    for (int bn = 64; bn <= 256; bn += 64) {
        const int64_t tiles = m_tiles * ((N + bn - 1) / bn), per_cu = bn == 64 ? 2 : 1, wgs = per_cu * LL_CUS;
        const double cost = (double)((tiles + wgs - 1) / wgs) * ll_cost(bn) * per_cu;
        if (best == 0 || cost <= least) {
            best = bn;
            least = cost;
        }
    }
    return best;
}

// Rows per tile of d hidden, whose sum is split over the columns until the CUs are full: the least work (backward pass for d
// hidden alone, 320 rows: 459 us with 192, 565 with 256 and 513 with 128; 576 rows 715, 876 and 825; 400 rows 628, 559, 599).
static int ll_dh_bn(int N) {
    int best = 64;
    for (int bn = 128; bn <= 256; bn += 64)
        if ((N + bn - 1) / bn * ll_cost(bn) <= (N + best - 1) / best * ll_cost(best)) best = bn;
    return best;
}

// Bytes in the order in which they are asked for, each on a multiple of 256.
struct LlLayout {
    size_t at = 0;
    size_t take(int64_t bytes) {
        const size_t begin = at;
        at += (size_t)ll_up(bytes, 256);
        return begin;
    }
};

// Rows up to which each workgroup counts those in front of it by itself (8192 rows of H = 2048: 31 us with the copy); more
// take a launch for it (20,000 rows: 24 us, the copy 33).  The counting does not depend on H, and hides behind the copy.
#define LL_COUNT_ROWS (1 << 14)
static int64_t ll_offsets_bytes(int N) { return N > LL_COUNT_ROWS ? (int64_t)((N + 15) / 16) * 4 : 0; }

struct LlForward {
    int bn, m_tiles, n_tiles, parts;
    int64_t n_pad;
    size_t plan, offsets, tok, row_of, hidden, partials, weighted, chosen, total;  // byte offsets, total size
};

static int ll_wm(int bn) {
    return bn == 64 ? MtShape<64>::WM : bn == 128 ? MtShape<128>::WM : bn == 192 ? MtShape<192>::WM : MtShape<256>::WM;
}

static LlForward ll_forward(int N, int H, int V, bool ent) {
    LlForward f;
    f.m_tiles = (V + MT_BM - 1) / MT_BM;
    f.bn = ll_bn(N, f.m_tiles);
    f.n_tiles = (N + f.bn - 1) / f.bn;
    f.parts = f.m_tiles * ll_wm(f.bn);
    f.n_pad = (int64_t)f.n_tiles * f.bn;
    LlLayout l;
    f.plan = l.take(8);
    f.offsets = l.take(ll_offsets_bytes(N));
    f.tok = l.take((int64_t)N * 4);
    f.row_of = l.take((int64_t)N * 4);
    f.hidden = l.take((int64_t)N * H * 2);
    f.partials = l.take(f.parts * f.n_pad * sizeof(float2));
    f.weighted = l.take(ent ? f.parts * f.n_pad * sizeof(float) : 0);
    f.chosen = l.take((int64_t)N * 4);
    f.total = l.at;
    return f;
}

struct LlBackward {
    int bn, n_tiles;           // of d logits
    int dh_bn, dh_tiles, h_tiles, splits, slab_rows;  // of d hidden
    int64_t n_pad;             // rows of G: whole steps of d weight
    int64_t chunk;             // columns of G: a multiple of 256
    int n_chunks;
    size_t plan, offsets, pos, rows, tok, hidden, copy, g, slabs, total;
};

static LlBackward ll_backward(int N, int H, int V, bool want_h, bool want_w) {
    LlBackward b;
    b.dh_bn = ll_dh_bn(N);
    b.dh_tiles = (N + b.dh_bn - 1) / b.dh_bn;
    b.h_tiles = (H + MT_BM - 1) / MT_BM;
    b.n_pad = ll_up(N, MT_BK);
    const int64_t v_pad = ll_up(V, MT_BM);
    int64_t most = LL_CHUNK_BYTES / 4 / b.n_pad / MT_BM * MT_BM;
    if (most < MT_BM) most = MT_BM;
    b.n_chunks = (int)((v_pad + most - 1) / most);
    b.chunk = ll_up((v_pad + b.n_chunks - 1) / b.n_chunks, MT_BM);
    b.n_chunks = (int)((v_pad + b.chunk - 1) / b.chunk);
    b.bn = ll_bn(N, b.chunk / MT_BM);
    b.n_tiles = (N + b.bn - 1) / b.bn;
    const int steps = (int)(b.chunk / MT_BK);
    b.splits = ll_splits(N, b.dh_bn, b.h_tiles, steps, 1 << 30);
    b.slab_rows = (int)ll_up(N, b.dh_bn) * b.splits;  // fewer rows take more splits, as far as this room goes
    LlLayout l;
    b.plan = l.take(8);
    b.offsets = l.take(ll_offsets_bytes(N));
    b.pos = l.take((int64_t)N * 4);
    b.rows = l.take((int64_t)N * sizeof(LlRow));
    b.tok = l.take((int64_t)N * 4);
    b.hidden = l.take((int64_t)N * H * 2);
    b.copy = l.take(want_w ? b.n_pad * H * 2 : 0);
    b.g = l.take(b.n_pad * b.chunk * 4);
    b.slabs = l.take(want_h ? (int64_t)b.slab_rows * H * 4 : 0);
    b.total = l.at;
    return b;
}

extern "C" size_t grx_lm_token_logps_scratch_bytes(int32_t N, int32_t H, int32_t V, int32_t entropy) {
    if (N <= 0 || V <= 0 || H <= 0 || N > GRX_MAX_TOKEN_ROWS || V > (1 << 24)) return 0;
    return ll_forward(N, H, V, entropy != 0).total;
}

extern "C" size_t grx_lm_token_logps_backward_scratch_bytes(int32_t N, int32_t H, int32_t V, int32_t want_hidden,
                                                            int32_t want_weight) {
    if (N <= 0 || V <= 0 || H <= 0 || N > GRX_MAX_TOKEN_ROWS || V > (1 << 24)) return 0;
    return ll_backward(N, H, V, want_hidden != 0, want_weight != 0).total;
}

extern "C" size_t grx_lm_token_logps_kept_bytes(int32_t N, int32_t V) {
    if (N <= 0 || V <= 0 || N > (1 << 20) || V > (1 << 24)) return 0;
    const LlForward f = ll_forward(N, 64, V, false);
    return (size_t)f.m_tiles * MT_BM * (size_t)f.n_pad * 4;
}

static int ll_check(const char* who, const grx_lm_token_logps_args* p) {
    GRX_REQUIRE(p != nullptr, GRX_E_INVALID, "%s: null args", who);
    GRX_REQUIRE(p->N >= 0 && p->V >= 1 && p->H >= 1, GRX_E_INVALID, "%s: bad shape", who);
    GRX_REQUIRE(p->H % 64 == 0, GRX_E_UNSUPPORTED, "%s: H must be a multiple of 64", who);
    GRX_REQUIRE(p->H <= (1 << 16) && p->V <= (1 << 24) && p->N <= GRX_MAX_TOKEN_ROWS, GRX_E_UNSUPPORTED,
                "%s: H above 2^16, V above 2^24 or more than %d rows", who, GRX_MAX_TOKEN_ROWS);
    // its inverse has to be finite too
    GRX_REQUIRE(p->temperature >= FLT_MIN && p->temperature < INFINITY, GRX_E_INVALID, "%s: temperature must be at least 2^-126", who);
    GRX_REQUIRE(p->hidden_stride >= p->H && p->weight_stride >= p->H && p->hidden_stride % 8 == 0 && p->weight_stride % 8 == 0,
                GRX_E_INVALID, "%s: operand rows must be 16-byte aligned and at least H long", who);
    GRX_REQUIRE(p->hidden_stride <= (1 << 22) && p->weight_stride <= (1 << 22), GRX_E_UNSUPPORTED,
                "%s: operand rows more than 2^22 elements apart", who);
    if (p->N == 0) return GRX_OK;
    GRX_REQUIRE(p->hidden != nullptr && p->weight != nullptr && p->token_ids != nullptr && p->row_stats != nullptr, GRX_E_INVALID,
                "%s: null buffer", who);
    GRX_REQUIRE((((uintptr_t)p->hidden | (uintptr_t)p->weight | (uintptr_t)p->kept) & 15u) == 0 && ((uintptr_t)p->row_stats & 7u) == 0, GRX_E_INVALID,
                "%s: misaligned buffer", who);
    GRX_REQUIRE(p->kept == nullptr || grx_lm_token_logps_kept_bytes(p->N, p->V) > 0, GRX_E_UNSUPPORTED,
                "%s: products are kept of up to 2^20 rows", who);
    return GRX_OK;
}

// Kernels that take more than 64 KB of LDS have to be told so, once per device.
template <typename K>
static int ll_allow_lds(K kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    GRX_CHECK_HIP(hipGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        GRX_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    return GRX_OK;
}

template <int BN, typename K, typename A>
static int ll_launch(K kernel, int64_t grid, const A& args, hipStream_t stream, std::atomic<uint64_t>& done) {
    const int rc = ll_allow_lds(kernel, mt_lds_bytes<BN>(), done);
    if (rc != GRX_OK) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(MtShape<BN>::THREADS), mt_lds_bytes<BN>(), stream, args);
    GRX_CHECK_HIP(hipGetLastError());
    return GRX_OK;
}

// Workgroups of a kernel that walks its tiles: as many as are resident (two per CU where the LDS holds two).
static int64_t ll_resident(int bn, int64_t tiles) {
    const int64_t most = bn == 64 ? 2 * LL_CUS : LL_CUS;
    return tiles < most ? tiles : most;
}

#define LL_ONE(BN, kernel, grid, args)                                     \
    do {                                                                   \
        static std::atomic<uint64_t> done_{0};                             \
        const int rc_ = ll_launch<BN>(kernel, grid, args, stream, done_);  \
        if (rc_ != GRX_OK) return rc_;                                     \
    } while (0)
#define LL_EACH(bn, kernel, grid, args)                     \
    do {                                                    \
        if ((bn) == 64) LL_ONE(64, (kernel<64>), grid, args);        \
        else if ((bn) == 128) LL_ONE(128, (kernel<128>), grid, args); \
        else if ((bn) == 192) LL_ONE(192, (kernel<192>), grid, args); \
        else LL_ONE(256, (kernel<256>), grid, args);        \
    } while (0)
#define LL_EACH_ENT(bn, ent, kernel, grid, args)                                  \
    do {                                                                          \
        if ((bn) == 64) {                                                         \
            if (ent) LL_ONE(64, (kernel<64, true>), grid, args);                  \
            else LL_ONE(64, (kernel<64, false>), grid, args);                     \
        } else if ((bn) == 128) {                                                 \
            if (ent) LL_ONE(128, (kernel<128, true>), grid, args);                \
            else LL_ONE(128, (kernel<128, false>), grid, args);                   \
        } else if ((bn) == 192) {                                                 \
            if (ent) LL_ONE(192, (kernel<192, true>), grid, args);                \
            else LL_ONE(192, (kernel<192, false>), grid, args);                   \
        } else {                                                                  \
            if (ent) LL_ONE(256, (kernel<256, true>), grid, args);                \
            else LL_ONE(256, (kernel<256, false>), grid, args);                   \
        }                                                                         \
    } while (0)

template <bool BACK>
static int ll_compact(LlCompact& c, const grx_lm_token_logps_args* p, int* offsets, hipStream_t stream) {
    c.hidden = reinterpret_cast<const uint16_t*>(p->hidden);
    c.hidden_ld = p->hidden_stride;
    c.ids = p->token_ids;
    c.N = p->N;
    c.H = p->H;
    c.V = p->V;
    c.stats = reinterpret_cast<float2*>(p->row_stats);
    c.entropy = p->entropy;
    const int blocks = (p->N + 15) / 16;
    if (p->N > LL_COUNT_ROWS) {
        hipLaunchKernelGGL(lm_logps_offsets_kernel<BACK>, dim3(1), dim3(1024), 0, stream, c, offsets, blocks);
        GRX_CHECK_HIP(hipGetLastError());
        c.offsets = offsets;
    }
    hipLaunchKernelGGL(lm_logps_compact_kernel<BACK>, dim3((unsigned)blocks, (unsigned)((p->H + 511) / 512)), dim3(256), 0, stream, c);
    GRX_CHECK_HIP(hipGetLastError());
    return GRX_OK;
}

extern "C" int grx_lm_token_logps(const grx_lm_token_logps_args* p, void* scratch, size_t scratch_bytes, void* stream_) {
    const char* who = "grx_lm_token_logps";
    const int rc = ll_check(who, p);
    if (rc != GRX_OK || p->N == 0) return rc;
    GRX_REQUIRE(p->logps != nullptr, GRX_E_INVALID, "%s: null logps", who);
    const bool ent = p->entropy != nullptr;
    const LlForward f = ll_forward(p->N, p->H, p->V, ent);
    GRX_REQUIRE(scratch != nullptr && scratch_bytes >= f.total, GRX_E_WORKSPACE, "%s: scratch of %zu bytes, need %zu", who,
                scratch_bytes, f.total);
    GRX_REQUIRE(((uintptr_t)scratch & 15u) == 0, GRX_E_INVALID, "%s: misaligned scratch", who);
    GRX_REQUIRE((int64_t)f.m_tiles * f.n_tiles < (1ll << 31) - LL_CUS * 2, GRX_E_UNSUPPORTED, "%s: too many tiles", who);
    hipStream_t stream = (hipStream_t)stream_;
    char* s = reinterpret_cast<char*>(scratch);
    LlCompact c = {};
    c.to = reinterpret_cast<uint16_t*>(s + f.hidden);
    c.plan = reinterpret_cast<int*>(s + f.plan);
    c.tok = reinterpret_cast<int*>(s + f.tok);
    c.row_of = reinterpret_cast<int*>(s + f.row_of);
    c.logps = p->logps;
    const int compact = ll_compact<false>(c, p, reinterpret_cast<int*>(s + f.offsets), stream);
    if (compact != GRX_OK) return compact;
    LlJoin j;
    LlArgs& a = j.g;
    a.o = {reinterpret_cast<const uint16_t*>(p->weight), p->weight_stride, c.to, c.plan, p->H, p->V};
    a.k = (float)(1.4426950408889634 / (double)p->temperature);
    a.tok = c.tok;
    a.partials = reinterpret_cast<float2*>(s + f.partials);
    a.weighted = ent ? reinterpret_cast<float*>(s + f.weighted) : nullptr;
    a.n_pad = f.n_pad;
    a.chosen = reinterpret_cast<float*>(s + f.chosen);
    a.m_tiles = f.m_tiles;
    a.kept = p->kept;
    const int64_t wgs = ll_resident(f.bn, (int64_t)a.m_tiles * f.n_tiles);
    if (p->kept) LL_EACH_ENT(f.bn, ent, lm_logps_keep_kernel, wgs, a);
    else LL_EACH_ENT(f.bn, ent, lm_logps_kernel, wgs, a);
    j.parts = f.parts;
    j.logps = p->logps;
    j.stats = reinterpret_cast<float2*>(p->row_stats);
    j.entropy = p->entropy;
    j.row_of = c.row_of;
    if (p->N <= 1024) hipLaunchKernelGGL(lm_logps_join_kernel<1>, dim3((unsigned)p->N), dim3(256), 0, stream, j);
    else hipLaunchKernelGGL(lm_logps_join_kernel<16>, dim3((unsigned)((p->N + 15) / 16)), dim3(256), 0, stream, j);
    GRX_CHECK_HIP(hipGetLastError());
    return GRX_OK;
}

extern "C" int grx_lm_token_logps_backward(const grx_lm_token_logps_args* p, void* scratch, size_t scratch_bytes,
                                           void* stream_) {
    const char* who = "grx_lm_token_logps_backward";
    const int rc = ll_check(who, p);
    if (rc != GRX_OK) return rc;
    GRX_REQUIRE(p->grad_entropy == nullptr || p->entropy != nullptr, GRX_E_INVALID,
                "%s: a gradient of the entropies needs the entropies", who);
    GRX_REQUIRE((((uintptr_t)p->grad_hidden | (uintptr_t)p->grad_weight) & 15u) == 0, GRX_E_INVALID, "%s: misaligned gradient", who);
    const bool want_h = p->grad_hidden != nullptr, want_w = p->grad_weight != nullptr, ent = p->grad_entropy != nullptr;
    if (p->N == 0 || (!want_h && !want_w)) return GRX_OK;
    const LlBackward b = ll_backward(p->N, p->H, p->V, want_h, want_w);
    GRX_REQUIRE(scratch != nullptr && scratch_bytes >= b.total, GRX_E_WORKSPACE, "%s: scratch of %zu bytes, need %zu", who,
                scratch_bytes, b.total);
    GRX_REQUIRE(((uintptr_t)scratch & 15u) == 0, GRX_E_INVALID, "%s: misaligned scratch", who);
    GRX_REQUIRE((int64_t)b.splits * b.h_tiles * b.dh_tiles < (1 << 23), GRX_E_UNSUPPORTED, "%s: too many tiles", who);
    GRX_REQUIRE((int64_t)p->N * p->H / 1024 < (1 << 24), GRX_E_UNSUPPORTED, "%s: more than 2^34 hidden elements", who);
    hipStream_t stream = (hipStream_t)stream_;
    char* s = reinterpret_cast<char*>(scratch);
    LlCompact k = {};
    k.to = reinterpret_cast<uint16_t*>(s + b.hidden);
    k.plan = reinterpret_cast<int*>(s + b.plan);
    k.tok = reinterpret_cast<int*>(s + b.tok);
    k.g = p->grad_logps;
    k.h = p->grad_entropy;
    k.inv_t = (float)(1.0 / (double)p->temperature);
    k.pos = reinterpret_cast<int*>(s + b.pos);
    k.rows = reinterpret_cast<LlRow*>(s + b.rows);
    k.dh_bn = b.dh_bn;
    k.h_tiles = b.h_tiles;
    k.steps = (int)(b.chunk / MT_BK);
    k.slab_rows = b.slab_rows;
    k.kept = p->kept != nullptr;
    const int compact = ll_compact<true>(k, p, reinterpret_cast<int*>(s + b.offsets), stream);
    if (compact != GRX_OK) return compact;
    const LlOperands o = {reinterpret_cast<const uint16_t*>(p->weight), p->weight_stride, k.to, k.plan, p->H, p->V};
    char* g = s + b.g;
    float* slabs = reinterpret_cast<float*>(s + b.slabs);
    if (want_w) {
        hipLaunchKernelGGL(lm_logps_prepare_kernel, dim3((unsigned)(b.n_pad / 64), (unsigned)(p->H / 32)), dim3(256), 0, stream, o, k.tok,
                           s + b.copy);
        GRX_CHECK_HIP(hipGetLastError());
    }
    for (int c = 0; c < b.n_chunks; ++c) {
        const int v0 = (int)(c * b.chunk), v64 = (int)(b.chunk / 64);
        const int64_t cols = ll_up(p->V - v0 < b.chunk ? p->V - v0 : b.chunk, MT_BM);
        LlGrad d = {o, (int)(cols / MT_BM), v0, v64, (float)(1.4426950408889634 / (double)p->temperature), k.rows, g};
        if (p->kept) {
            const int n32s = (int)(ll_forward(p->N, p->H, p->V, false).n_pad / 32);
            const dim3 grid((unsigned)(d.m_tiles * 2), (unsigned)(b.n_pad / 32));
            if (ent) hipLaunchKernelGGL(lm_logps_kept_kernel<true>, grid, dim3(256), 0, stream, d, p->kept, n32s);
            else hipLaunchKernelGGL(lm_logps_kept_kernel<false>, grid, dim3(256), 0, stream, d, p->kept, n32s);
            GRX_CHECK_HIP(hipGetLastError());
        } else {
            LL_EACH_ENT(b.bn, ent, lm_logps_dlogits_kernel, ll_resident(b.bn, (int64_t)d.m_tiles * b.n_tiles), d);
        }
        if (want_h) {
            LlDh x = {o, g, b.h_tiles, (int)(cols / MT_BK), v0, v64, c > 0, slabs};
            LL_EACH(b.dh_bn, lm_logps_dhidden_kernel, std::max<int64_t>((int64_t)b.splits * b.h_tiles * b.dh_tiles, LL_CUS), x);
        }
        if (want_w) {
            LlDw x = {s + b.copy, g, p->H, p->V, b.h_tiles, (int)(cols / 256), v0, v64, k.plan,
                      reinterpret_cast<uint16_t*>(p->grad_weight)};
            const int64_t wgs = ll_resident(256, (int64_t)x.m_tiles * x.n_tiles);
            if (b.n_pad / MT_BK * 2 <= LL_LINES_STEPS) LL_ONE(256, lm_logps_dweight_kernel<true>, wgs, x);
            else LL_ONE(256, lm_logps_dweight_kernel<false>, wgs, x);
        }
    }
    if (want_h) {
        const int64_t n = (int64_t)p->N * p->H;
        hipLaunchKernelGGL(lm_logps_dhidden_join_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, stream, o, p->N, slabs,
                           k.pos, reinterpret_cast<uint16_t*>(p->grad_hidden));
        GRX_CHECK_HIP(hipGetLastError());
    }
    return GRX_OK;
}
