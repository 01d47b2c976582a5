// Log-probabilities and entropies of tokens from hidden states [N, H] and the output projection [V, H], without
// logits: what token_logps.hip computes from them.  Forward, the products of a 256 x BN tile are consumed where they
// are: a row keeps (max, sum of exponentials, weighted sum) per 256 columns and its own token's logit.  Backward,
// the product is formed again and turned into the logits' gradient G = dL/dlogits in bf16 -- the type autograd would
// hold it in; half a step (2^-9) of each element, independent over the vocabulary -- in chunks of columns, and
//   d hidden = G x weight (sum over v),    d weight = G^T x hidden (sum over rows)
// follow with fp32 accumulators.  Four products of 2 N V H; bound by the matrix cores at many rows, by the weight
// (V H elements read per product, written once) at few.
#include <hip/hip_runtime.h>
#include <math.h>

#include <atomic>

#include "common.h"
#include "lse_math.h"
#include "mfma_tile.h"

#define LL_FLOOR (-200.f)
#define LL_CHUNK_BYTES (1ll << 30)  // G of one chunk

struct LlArgs {
    MtOperand w, h;             // weight [V, H], hidden [N, H]
    int N, H, V;
    int m_tiles, n_tiles;
    float k;                    // log2(e) / temperature
    const int64_t* ids;         // [N]
    float2* partials;           // [m_tiles][n_pad] (max, sum)
    float* weighted;            // [m_tiles][n_pad], with entropies
    int64_t n_pad;
    float* chosen;              // [N] logit of the row's token
};

template <int BN>
__global__ __launch_bounds__(MT_THREADS) void lm_logps_kernel(LlArgs a) {
    typedef MtShape<BN> S;
    extern __shared__ __align__(16) unsigned char lds[];
    int tm, tn;
    mt_tile(blockIdx.x, a.m_tiles, a.n_tiles, tm, tn);
    const int v0 = tm * MT_BM, r0 = tn * BN;
    mt_f32x16 acc[S::MA][S::NB];
    mt_multiply<BN, false, false>(acc, lds, a.w, v0, a.h, r0, 0, a.H / MT_BK);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN, half = lane >> 5;
    float* red = reinterpret_cast<float*>(lds);  // [3][WM][BN]
    const bool ent = a.weighted != nullptr;
#pragma unroll
    for (int n = 0; n < S::NB; ++n) {
        const int in_tile = wn * S::NB * 32 + n * 32 + (lane & 31);
        const int r = r0 + in_tile;
        float mx = -INFINITY;
        const int vw = v0 + wm * S::MA * 32 + 4 * half;  // vocabulary entry of m = 0, e = 0
#pragma unroll
        for (int m = 0; m < S::MA; ++m)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (vw + m * 32 + (e & 3) + 8 * (e >> 2) >= a.V) acc[m][n][e] = -INFINITY;
                mx = fmaxf(mx, acc[m][n][e]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));  // the other half of the lanes holds the same row
        const float ref = mx == -INFINITY ? 0.f : mx;
        float s = 0.f, u = 0.f;
#pragma unroll
        for (int m = 0; m < S::MA; ++m)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float t = (acc[m][n][e] - ref) * a.k;
                const float w = fast_exp2(t);
                s += w;
                if (ent) u = fmaf(w, fmaxf(t, LL_FLOOR), u);
            }
        s += __shfl_xor(s, 32, 64);
        u += __shfl_xor(u, 32, 64);
        if (half == 0) {
            red[wm * BN + in_tile] = mx;
            red[(S::WM + wm) * BN + in_tile] = s;
            red[(2 * S::WM + wm) * BN + in_tile] = u;
        }
        const int64_t id = r < a.N ? a.ids[r] : -1;
        const int64_t off = id - vw;  // 4 consecutive entries, every 8
        if (off >= 0 && off < S::MA * 32 && (off & 4) == 0) {
            const int at = (int)(off >> 5) * 16 + (int)((off & 31) >> 3) * 4 + (int)(off & 3);
#pragma unroll
            for (int m = 0; m < S::MA; ++m)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (m * 16 + e == at) a.chosen[r] = acc[m][n][e];
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < BN) {
        const int i = threadIdx.x;
        float m = red[i];
#pragma unroll
        for (int w = 1; w < S::WM; ++w) m = fmaxf(m, red[w * BN + i]);
        const float ref = m == -INFINITY ? 0.f : m;
        float s = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < S::WM; ++w) {
            const float d = fmaxf((red[w * BN + i] - ref) * a.k, LL_FLOOR), f = fast_exp2(d), sw = red[(S::WM + w) * BN + i];
            s = fmaf(sw, f, s);
            u += (red[(2 * S::WM + w) * BN + i] + sw * d) * f;
        }
        a.partials[(int64_t)tm * a.n_pad + r0 + i] = make_float2(m, s);
        if (ent) a.weighted[(int64_t)tm * a.n_pad + r0 + i] = u;
    }
}

struct LlJoin {
    LlArgs g;
    float* logps;
    float2* stats;
    float* entropy;
};

// Joins a row's column tiles: 16 rows per workgroup, 16 threads a row.
__global__ __launch_bounds__(256) void lm_logps_join_kernel(LlJoin a) {
    __shared__ float sm[16][17], ss[16][17], su[16][17];
    const int i = threadIdx.x & 15, j = threadIdx.x >> 4;
    const int r = blockIdx.x * 16 + i;
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
    for (int t = j; t < a.g.m_tiles; t += 16) {  // n_pad is a multiple of 64: rows past N read what a clamped row left
        const float2 p = a.g.partials[(int64_t)t * a.g.n_pad + r];
        add(p.x, p.y, a.entropy ? a.g.weighted[(int64_t)t * a.g.n_pad + r] : 0.f);
    }
    sm[j][i] = m;
    ss[j][i] = s;
    su[j][i] = u;
    __syncthreads();
    if (j != 0 || r >= a.g.N) return;
    for (int w = 1; w < 16; ++w) add(sm[w][i], ss[w][i], su[w][i]);
    const int64_t id = a.g.ids[r];
    const float ln2 = 0.69314718055994531f;
    const float ls = log2f(s);
    if (id < 0) {
        a.logps[r] = 0.f;
        a.stats[r] = make_float2(0.f, 1.f);
        if (a.entropy) a.entropy[r] = 0.f;
        return;
    }
    a.logps[r] = id < a.g.V ? ((a.g.chosen[r] - m) * k - ls) * ln2 : NAN;
    a.stats[r] = make_float2(m, s);
    if (a.entropy) a.entropy[r] = (ls - u / s) * ln2;
}

// ---- backward -----------------------------------------------------------------------------------------
// What a row needs to turn a product into its gradient: w = 2^((x - m) k), G = w (alpha + beta (x - m) k) + at at the
// token.  tok = -1: nothing flows into this row (padding, or both gradients 0); its G is 0 whatever the products are.
struct LlRow {
    float m, alpha, beta, at;
    int tok;
    int pad[3];
};

struct LlPrep {
    const int64_t* ids;
    const float2* stats;
    const float* entropy;
    const float* g;
    const float* h;
    float inv_t;
    int N, V, H;
    LlRow* rows;               // [n_pad]
    const uint16_t* hidden;
    int64_t hidden_ld;
    uint16_t* copy;            // [n_pad][H]: hidden with 0 in the rows that do not count; null: not needed
};

__global__ __launch_bounds__(256) void lm_logps_prepare_kernel(LlPrep a) {
    const int r = blockIdx.x;
    float g = 0.f, h = 0.f;
    int64_t id = -1;
    if (r < a.N) {
        id = a.ids[r];
        if (id >= 0) {
            g = a.g ? a.g[r] : 0.f;
            h = a.h ? a.h[r] : 0.f;
        }
    }
    const bool live = g != 0.f || h != 0.f;
    if (threadIdx.x == 0) {
        LlRow o = {0.f, 0.f, 0.f, 0.f, -1, {0, 0, 0}};
        if (live) {
            const float2 st = a.stats[r];
            const float ln2 = 0.69314718055994531f;
            o.m = st.x;
            o.alpha = -(g + (a.h ? h * (a.entropy[r] - log2f(st.y) * ln2) : 0.f)) * a.inv_t / st.y;
            o.beta = -h * ln2 * a.inv_t / st.y;
            o.at = id < a.V ? g * a.inv_t : NAN;
            if (id >= a.V) o.alpha = NAN;
            o.tok = id < a.V ? (int)id : 0;
        }
        a.rows[r] = o;
    }
    if (a.copy) {
        uint4* d = reinterpret_cast<uint4*>(a.copy + (int64_t)r * a.H);
        const uint4* s = reinterpret_cast<const uint4*>(a.hidden + (int64_t)r * a.hidden_ld);
        for (int i = threadIdx.x; i < a.H / 8; i += 256) d[i] = live ? s[i] : make_uint4(0, 0, 0, 0);
    }
}

struct LlGrad {
    MtOperand w, h;
    int N, H, V;
    int m_tiles, n_tiles;
    int v_begin;               // first column of the chunk
    float k;
    const LlRow* rows;
    uint16_t* out;             // [n_pad][ld]
    int64_t ld;
    int n_pad;
};

template <int BN>
__global__ __launch_bounds__(MT_THREADS) void lm_logps_dlogits_kernel(LlGrad a) {
    typedef MtShape<BN> S;
    extern __shared__ __align__(16) unsigned char lds[];
    int tm, tn;
    mt_tile(blockIdx.x, a.m_tiles, a.n_tiles, tm, tn);
    const int c0 = tm * MT_BM, v0 = a.v_begin + c0, r0 = tn * BN;
    mt_f32x16 acc[S::MA][S::NB];
    mt_multiply<BN, false, false>(acc, lds, a.w, v0, a.h, r0, 0, a.H / MT_BK);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN, half = lane >> 5;
#pragma unroll
    for (int n = 0; n < S::NB; ++n) {
        const int r = r0 + wn * S::NB * 32 + n * 32 + (lane & 31);
        if (r >= a.n_pad) continue;
        const LlRow row = a.rows[r];
        uint16_t* out = a.out + (int64_t)r * a.ld + c0 + wm * S::MA * 32 + 4 * half;
        const int vw = v0 + wm * S::MA * 32 + 4 * half;
        const int tok = row.tok - vw;
#pragma unroll
        for (int m = 0; m < S::MA; ++m)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                mt_f32x4 d;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int off = m * 32 + 8 * q + j;
                    const float t = (acc[m][n][q * 4 + j] - row.m) * a.k;
                    float v = fast_exp2(t) * fmaf(row.beta, fmaxf(t, LL_FLOOR), row.alpha);
                    if (off == tok) v += row.at;
                    d[j] = row.tok >= 0 && vw + off < a.V ? v : 0.f;
                }
                *reinterpret_cast<mt_b16x4*>(out + m * 32 + 8 * q) = __builtin_convertvector(d, mt_b16x4);
            }
    }
}

// d hidden: C[n][h] = sum over the chunk's columns of G[n][v] weight[v][h], fp32 slabs, one per split of the columns.
struct LlDh {
    MtOperand w, g;            // weight rows of the chunk (k across), G (k along)
    int N, H;
    int m_tiles, n_tiles, splits, steps, steps_per;
    int add;                   // 1: add to what the chunk before left
    float* slabs;              // [splits][N][H]
};

template <int BN>
__global__ __launch_bounds__(MT_THREADS) void lm_logps_dhidden_kernel(LlDh a) {
    typedef MtShape<BN> S;
    extern __shared__ __align__(16) unsigned char lds[];
    const int split = blockIdx.x % a.splits, tile = blockIdx.x / a.splits;
    const int tm = tile % a.m_tiles, tn = tile / a.m_tiles;
    const int h0 = tm * MT_BM, r0 = tn * BN;
    const int s0 = split * a.steps_per, s1 = s0 + a.steps_per < a.steps ? s0 + a.steps_per : a.steps;
    mt_f32x16 acc[S::MA][S::NB];
    mt_multiply<BN, true, false>(acc, lds, a.w, h0, a.g, r0, s0 * MT_BK, s1 - s0);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN, half = lane >> 5;
    float* slab = a.slabs + (int64_t)split * a.N * a.H;
#pragma unroll
    for (int n = 0; n < S::NB; ++n) {
        const int r = r0 + wn * S::NB * 32 + n * 32 + (lane & 31);
        if (r >= a.N) continue;
#pragma unroll
        for (int m = 0; m < S::MA; ++m)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int h = h0 + wm * S::MA * 32 + m * 32 + 8 * q + 4 * half;
                if (h >= a.H) continue;
                mt_f32x4* o = reinterpret_cast<mt_f32x4*>(slab + (int64_t)r * a.H + h);
                mt_f32x4 v = {acc[m][n][q * 4], acc[m][n][q * 4 + 1], acc[m][n][q * 4 + 2], acc[m][n][q * 4 + 3]};
                if (a.add) v += *o;
                *o = v;
            }
    }
}

// Sum of the slabs in their order, rounded once.
__global__ __launch_bounds__(256) void lm_logps_dhidden_join_kernel(const float* slabs, int splits, int64_t n, int H,
                                                                    const LlRow* rows, uint16_t* out) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    mt_f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (rows[i / H].tok >= 0)
        for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const mt_f32x4*>(slabs + s * n + i);
    *reinterpret_cast<mt_b16x4*>(out + i) = __builtin_convertvector(v, mt_b16x4);
}

// d weight of the chunk: C[v][h] = sum over the rows of G[n][v] hidden[n][h].
struct LlDw {
    MtOperand h, g;            // hidden copy (k across), G (k across)
    int H, V;
    int m_tiles, n_tiles, steps;
    int v_begin;
    uint16_t* out;             // [V][H]
};

__global__ __launch_bounds__(MT_THREADS) void lm_logps_dweight_kernel(LlDw a) {
    typedef MtShape<256> S;
    extern __shared__ __align__(16) unsigned char lds[];
    int tm, tn;
    mt_tile(blockIdx.x, a.m_tiles, a.n_tiles, tm, tn);
    const int h0 = tm * MT_BM, c0 = tn * 256;
    mt_f32x16 acc[S::MA][S::NB];
    mt_multiply<256, true, true>(acc, lds, a.h, h0, a.g, c0, 0, a.steps);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / S::WN, wn = wave % S::WN, half = lane >> 5;
#pragma unroll
    for (int n = 0; n < S::NB; ++n) {
        const int v = a.v_begin + c0 + wn * S::NB * 32 + n * 32 + (lane & 31);
        if (v >= a.V) continue;
#pragma unroll
        for (int m = 0; m < S::MA; ++m)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int h = h0 + wm * S::MA * 32 + m * 32 + 8 * q + 4 * half;
                if (h >= a.H) continue;
                const mt_f32x4 x = {acc[m][n][q * 4], acc[m][n][q * 4 + 1], acc[m][n][q * 4 + 2], acc[m][n][q * 4 + 3]};
                *reinterpret_cast<mt_b16x4*>(a.out + (int64_t)v * a.H + h) = __builtin_convertvector(x, mt_b16x4);
            }
    }
}

// ---- host ------------------------------------------------------------------------------------------
static int64_t ll_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// Rows per tile: as few as hold all rows.
static int ll_bn(int N) { return N <= 64 ? 64 : N <= 128 ? 128 : 256; }

struct LlForward {
    int bn, m_tiles, n_tiles;
    int64_t n_pad;
    size_t partials, weighted, chosen, total;  // byte offsets, total size
};

static LlForward ll_forward(int N, int V, bool ent) {
    LlForward f;
    f.bn = ll_bn(N);
    f.m_tiles = (V + MT_BM - 1) / MT_BM;
    f.n_tiles = (N + f.bn - 1) / f.bn;
    f.n_pad = (int64_t)f.n_tiles * f.bn;
    f.partials = 0;
    f.weighted = (size_t)f.m_tiles * f.n_pad * sizeof(float2);
    f.chosen = f.weighted + (ent ? (size_t)f.m_tiles * f.n_pad * sizeof(float) : 0);
    f.total = f.chosen + (size_t)N * sizeof(float);
    return f;
}

struct LlBackward {
    int bn, n_tiles, h_tiles;
    int64_t n_pad;             // rows of G: a multiple of 64, the step of d weight's sum
    int64_t chunk;             // columns of G: a multiple of 256
    int n_chunks;
    int splits;
    size_t rows, copy, g, slabs, total;
};

// Splits of d hidden's sum: as many as fill the 256 CUs evenly, each at least eight steps long.
static int ll_splits(int tiles, int64_t steps) {
    int best = 1;
    double best_use = 0.0;
    for (int s = 1; s <= 64 && (s == 1 || steps / s >= 8); ++s) {
        const int64_t wgs = (int64_t)tiles * s;
        const double use = (double)wgs / (double)(ll_up(wgs, 256));
        if (use > best_use + 0.04) {
            best_use = use;
            best = s;
        }
    }
    return best;
}

static LlBackward ll_backward(int N, int H, int V, bool want_h, bool want_w) {
    LlBackward b;
    b.bn = ll_bn(N);
    b.n_tiles = (N + b.bn - 1) / b.bn;
    b.h_tiles = (H + MT_BM - 1) / MT_BM;
    b.n_pad = ll_up(N, MT_BK);
    const int64_t v_pad = ll_up(V, MT_BM);
    int64_t most = LL_CHUNK_BYTES / 2 / b.n_pad / MT_BM * MT_BM;
    if (most < MT_BM) most = MT_BM;
    b.n_chunks = (int)((v_pad + most - 1) / most);
    b.chunk = ll_up((v_pad + b.n_chunks - 1) / b.n_chunks, MT_BM);
    b.n_chunks = (int)((v_pad + b.chunk - 1) / b.chunk);
    b.splits = ll_splits(b.h_tiles * b.n_tiles, b.chunk / MT_BK);
    b.rows = 0;
    b.copy = (size_t)ll_up(b.n_pad * sizeof(LlRow), 256);
    b.g = b.copy + (want_w ? (size_t)ll_up(b.n_pad * H * 2, 256) : 0);
    b.slabs = b.g + (size_t)ll_up(b.n_pad * b.chunk * 2, 256);
    b.total = b.slabs + (want_h ? (size_t)b.splits * N * H * sizeof(float) : 0);
    return b;
}

extern "C" size_t grx_lm_token_logps_scratch_bytes(int32_t N, int32_t H, int32_t V, int32_t entropy) {
    if (N <= 0 || V <= 0 || H <= 0 || N > GRX_MAX_TOKEN_ROWS || V > (1 << 24)) return 0;
    return ll_forward(N, V, entropy != 0).total;
}

extern "C" size_t grx_lm_token_logps_backward_scratch_bytes(int32_t N, int32_t H, int32_t V, int32_t want_hidden,
                                                            int32_t want_weight) {
    if (N <= 0 || V <= 0 || H <= 0 || N > GRX_MAX_TOKEN_ROWS || V > (1 << 24)) return 0;
    return ll_backward(N, H, V, want_hidden != 0, want_weight != 0).total;
}

static int ll_check(const char* who, const grx_lm_token_logps_args* p) {
    GRX_REQUIRE(p != nullptr, GRX_E_INVALID, "%s: null args", who);
    GRX_REQUIRE(p->N >= 0 && p->V >= 1 && p->H >= 1, GRX_E_INVALID, "%s: bad shape", who);
    GRX_REQUIRE(p->H % 64 == 0, GRX_E_UNSUPPORTED, "%s: H must be a multiple of 64", who);
    GRX_REQUIRE(p->H <= (1 << 16) && p->V <= (1 << 24) && p->N <= GRX_MAX_TOKEN_ROWS, GRX_E_UNSUPPORTED,
                "%s: H above 2^16, V above 2^24 or more than %d rows", who, GRX_MAX_TOKEN_ROWS);
    GRX_REQUIRE(p->temperature > 0.f && p->temperature < INFINITY, GRX_E_INVALID, "%s: temperature must be positive", who);
    GRX_REQUIRE(p->hidden_stride >= p->H && p->weight_stride >= p->H && p->hidden_stride % 8 == 0 && p->weight_stride % 8 == 0,
                GRX_E_INVALID, "%s: operand rows must be 16-byte aligned and at least H long", who);
    if (p->N == 0) return GRX_OK;
    GRX_REQUIRE(p->hidden != nullptr && p->weight != nullptr && p->token_ids != nullptr && p->row_stats != nullptr, GRX_E_INVALID,
                "%s: null buffer", who);
    GRX_REQUIRE((((uintptr_t)p->hidden | (uintptr_t)p->weight) & 15u) == 0 && ((uintptr_t)p->row_stats & 7u) == 0, GRX_E_INVALID,
                "%s: misaligned buffer", who);
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

#define LL_LAUNCH(kernel, BN, grid, args)                                                                       \
    do {                                                                                                        \
        static std::atomic<uint64_t> done_{0};                                                                  \
        const int rc_ = ll_allow_lds(kernel, mt_lds_bytes<BN>(), done_);                                        \
        if (rc_ != GRX_OK) return rc_;                                                                          \
        hipLaunchKernelGGL(kernel, dim3((unsigned)(grid)), dim3(MT_THREADS), mt_lds_bytes<BN>(), stream, args); \
        GRX_CHECK_HIP(hipGetLastError());                                                                       \
    } while (0)

#define LL_LAUNCH_BN(kernel, bn, grid, args)                        \
    do {                                                            \
        if ((bn) == 64) LL_LAUNCH((kernel<64>), 64, grid, args);    \
        else if ((bn) == 128) LL_LAUNCH((kernel<128>), 128, grid, args); \
        else LL_LAUNCH((kernel<256>), 256, grid, args);             \
    } while (0)

extern "C" int grx_lm_token_logps(const grx_lm_token_logps_args* p, void* scratch, size_t scratch_bytes, void* stream_) {
    const char* who = "grx_lm_token_logps";
    int rc = ll_check(who, p);
    if (rc != GRX_OK || p->N == 0) return rc;
    GRX_REQUIRE(p->logps != nullptr, GRX_E_INVALID, "%s: null logps", who);
    const LlForward f = ll_forward(p->N, p->V, p->entropy != nullptr);
    GRX_REQUIRE(scratch != nullptr && scratch_bytes >= f.total, GRX_E_WORKSPACE, "%s: scratch of %zu bytes, need %zu", who,
                scratch_bytes, f.total);
    GRX_REQUIRE(((uintptr_t)scratch & 15u) == 0, GRX_E_INVALID, "%s: misaligned scratch", who);
    GRX_REQUIRE((int64_t)f.m_tiles * f.n_tiles < (1 << 23), GRX_E_UNSUPPORTED, "%s: too many tiles", who);
    hipStream_t stream = (hipStream_t)stream_;
    char* s = reinterpret_cast<char*>(scratch);
    LlJoin j;
    LlArgs& a = j.g;
    a.w = {reinterpret_cast<const uint16_t*>(p->weight), p->weight_stride, p->V, 0};
    a.h = {reinterpret_cast<const uint16_t*>(p->hidden), p->hidden_stride, p->N, 0};
    a.N = p->N;
    a.H = p->H;
    a.V = p->V;
    a.m_tiles = f.m_tiles;
    a.n_tiles = f.n_tiles;
    a.k = (float)(1.4426950408889634 / (double)p->temperature);
    a.ids = p->token_ids;
    a.partials = reinterpret_cast<float2*>(s + f.partials);
    a.weighted = p->entropy ? reinterpret_cast<float*>(s + f.weighted) : nullptr;
    a.n_pad = f.n_pad;
    a.chosen = reinterpret_cast<float*>(s + f.chosen);
    LL_LAUNCH_BN(lm_logps_kernel, f.bn, f.m_tiles * f.n_tiles, a);
    j.logps = p->logps;
    j.stats = reinterpret_cast<float2*>(p->row_stats);
    j.entropy = p->entropy;
    hipLaunchKernelGGL(lm_logps_join_kernel, dim3((unsigned)((p->N + 15) / 16)), dim3(256), 0, stream, j);
    GRX_CHECK_HIP(hipGetLastError());
    return GRX_OK;
}

extern "C" int grx_lm_token_logps_backward(const grx_lm_token_logps_args* p, void* scratch, size_t scratch_bytes,
                                           void* stream_) {
    const char* who = "grx_lm_token_logps_backward";
    int rc = ll_check(who, p);
    if (rc != GRX_OK) return rc;
    GRX_REQUIRE(p->grad_entropy == nullptr || p->entropy != nullptr, GRX_E_INVALID,
                "%s: a gradient of the entropies needs the entropies", who);
    GRX_REQUIRE((((uintptr_t)p->grad_hidden | (uintptr_t)p->grad_weight) & 15u) == 0, GRX_E_INVALID, "%s: misaligned gradient", who);
    const bool want_h = p->grad_hidden != nullptr, want_w = p->grad_weight != nullptr;
    if (p->N == 0 || (!want_h && !want_w)) return GRX_OK;
    const LlBackward b = ll_backward(p->N, p->H, p->V, want_h, want_w);
    GRX_REQUIRE(scratch != nullptr && scratch_bytes >= b.total, GRX_E_WORKSPACE, "%s: scratch of %zu bytes, need %zu", who,
                scratch_bytes, b.total);
    GRX_REQUIRE(((uintptr_t)scratch & 15u) == 0, GRX_E_INVALID, "%s: misaligned scratch", who);
    GRX_REQUIRE(b.chunk / MT_BM * b.n_tiles < (1 << 23) && (int64_t)b.splits * b.h_tiles * b.n_tiles < (1 << 23) &&
                    b.n_pad <= GRX_MAX_TOKEN_ROWS,
                GRX_E_UNSUPPORTED, "%s: too many tiles", who);
    hipStream_t stream = (hipStream_t)stream_;
    char* s = reinterpret_cast<char*>(scratch);
    LlRow* rows = reinterpret_cast<LlRow*>(s + b.rows);
    uint16_t* copy = want_w ? reinterpret_cast<uint16_t*>(s + b.copy) : nullptr;
    uint16_t* g = reinterpret_cast<uint16_t*>(s + b.g);
    float* slabs = reinterpret_cast<float*>(s + b.slabs);
    const uint16_t* weight = reinterpret_cast<const uint16_t*>(p->weight);
    const uint16_t* hidden = reinterpret_cast<const uint16_t*>(p->hidden);

    LlPrep pr = {p->token_ids, reinterpret_cast<const float2*>(p->row_stats), p->entropy, p->grad_logps, p->grad_entropy,
                 (float)(1.0 / (double)p->temperature), p->N, p->V, p->H, rows, hidden, p->hidden_stride, copy};
    hipLaunchKernelGGL(lm_logps_prepare_kernel, dim3((unsigned)b.n_pad), dim3(256), 0, stream, pr);
    GRX_CHECK_HIP(hipGetLastError());
    for (int c = 0; c < b.n_chunks; ++c) {
        const int v0 = (int)(c * b.chunk);
        const int64_t cols = ll_up(p->V - v0 < b.chunk ? p->V - v0 : b.chunk, MT_BM);
        LlGrad d = {{weight, p->weight_stride, p->V, 0}, {hidden, p->hidden_stride, p->N, 0}, p->N, p->H, p->V,
                    (int)(cols / MT_BM), b.n_tiles, v0, (float)(1.4426950408889634 / (double)p->temperature), rows, g, b.chunk,
                    (int)b.n_pad};
        LL_LAUNCH_BN(lm_logps_dlogits_kernel, b.bn, d.m_tiles * d.n_tiles, d);
        if (want_h) {
            LlDh x;
            x.w = {weight + (int64_t)v0 * p->weight_stride, p->weight_stride, p->H, p->V - v0};
            x.g = {g, b.chunk, (int)b.n_pad, 0};
            x.N = p->N;
            x.H = p->H;
            x.m_tiles = b.h_tiles;
            x.n_tiles = b.n_tiles;
            x.splits = b.splits;
            x.steps = (int)(cols / MT_BK);
            x.steps_per = (x.steps + b.splits - 1) / b.splits;
            x.add = c > 0;
            x.slabs = slabs;
            LL_LAUNCH_BN(lm_logps_dhidden_kernel, b.bn, b.splits * b.h_tiles * b.n_tiles, x);
        }
        if (want_w) {
            LlDw x;
            x.h = {copy, p->H, p->H, (int)b.n_pad};
            x.g = {g, b.chunk, (int)cols, (int)b.n_pad};
            x.H = p->H;
            x.V = p->V;
            x.m_tiles = b.h_tiles;
            x.n_tiles = (int)(cols / 256);
            x.steps = (int)(b.n_pad / MT_BK);
            x.v_begin = v0;
            x.out = reinterpret_cast<uint16_t*>(p->grad_weight);
            LL_LAUNCH(lm_logps_dweight_kernel, 256, x.m_tiles * x.n_tiles, x);
        }
    }
    if (want_h) {
        const int64_t n = (int64_t)p->N * p->H;
        hipLaunchKernelGGL(lm_logps_dhidden_join_kernel, dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, stream, slabs, b.splits,
                           n, p->H, rows, reinterpret_cast<uint16_t*>(p->grad_hidden));
        GRX_CHECK_HIP(hipGetLastError());
    }
    return GRX_OK;
}
