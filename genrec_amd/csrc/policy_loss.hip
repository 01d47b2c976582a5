// Clipped policy loss with a KL term, and its gradient, on per-token log-probabilities.  Per valid token, with
// d = logp - old (or its mean over the row's valid tokens: one ratio per sequence), w = exp(d), A the advantage:
//   l = -min(min(w, delta) A, clip(w, 1 - e_low, 1 + e_high) A) + beta (exp(q) - 1 - q),      q = ref - logp
//   dl/dlogp = -w A where the clipped term is not the smaller one, + -beta (exp(q) - 1)
// and the loss is the sum of l under one of four weights: 1 / (rows x tokens of the row), 1 / tokens of the batch,
// or a constant.  About 20 bytes a token; a launcher's batch is 320 tokens, so small calls are launch latency (one
// workgroup, one launch) and large ones HBM.
//
// Differences are taken, and compared with log(1 - e_low), log(1 + e_high), log(delta), in 64 bits: which side of a
// bound a token is on does not depend on the rounding of exp.  Terms are fp32, all sums 64 bits, in a fixed order.
#include <hip/hip_runtime.h>
#include <math.h>
#include <string.h>

#include "common.h"

#define PL_THREADS 256
#define PL_BIG 1024
#define PL_SINGLE_TOKENS 4096   // up to here one workgroup does the whole call
#define PL_MAX_WGS 2048
#define PL_SUMS 5               // loss, kl, clipped below, clipped above, valid tokens

struct PlArgs {
    grx_policy_loss_args p;
    double log_low, log_high, log_delta;
    float low, high, delta;
    double constant;            // the weight all tokens share; 0: 1 / valid tokens of the batch
    double* partials;           // [gridDim][PL_SUMS]; null: this launch is one workgroup and finishes the call
    int n_partials;
};

__device__ __forceinline__ bool pl_valid(const grx_policy_loss_args& p, int64_t r, int t) {
    const int64_t i = r * p.mask_stride + t;
    switch (p.mask_type) {
        case GRX_MASK_U8: return static_cast<const uint8_t*>(p.mask)[i] != 0;
        case GRX_MASK_I32: return static_cast<const int32_t*>(p.mask)[i] > 0;
        case GRX_MASK_I64: return static_cast<const int64_t*>(p.mask)[i] > 0;
        default: return static_cast<const float*>(p.mask)[i] > 0.f;
    }
}

// exp(q) - 1 - q without the cancellation near 0: its Taylor series (the first term left out is below 2^-26 of the
// sum for |q| < 1), the difference itself elsewhere.  rise: exp(q) - 1, which stays finite where q = -inf.
__device__ __forceinline__ float pl_kl(float q, float& rise) {
    if (fabsf(q) < 1.f) {
        float s = 1.f / 39916800.f;
        s = fmaf(s, q, 1.f / 3628800.f);
        s = fmaf(s, q, 1.f / 362880.f);
        s = fmaf(s, q, 1.f / 40320.f);
        s = fmaf(s, q, 1.f / 5040.f);
        s = fmaf(s, q, 1.f / 720.f);
        s = fmaf(s, q, 1.f / 120.f);
        s = fmaf(s, q, 1.f / 24.f);
        s = fmaf(s, q, 1.f / 6.f);
        s = fmaf(s, q, 0.5f);
        const float kl = s * q * q;
        rise = kl + q;
        return kl;
    }
    rise = expf(q) - 1.f;
    return rise - q;
}

// Sum over the LANES lanes that share a row; every lane gets it.  LANES > 64: a whole workgroup.
template <int LANES>
__device__ __forceinline__ double pl_row_sum(double v, double* lds) {
#pragma unroll
    for (int o = (LANES < 64 ? LANES : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int w = 0; w < LANES / 64; ++w) v += lds[w];
    }
    return v;
}

struct PlTerm {
    float loss, slope, kl, kl_slope;
    bool cut_low, cut_high;
};

// A thread's share of the sums; loss: of its present row, without the row's weight.
struct PlShare {
    double total, loss, kl;
    int low, high, valid;
};

// One token: d = log ratio in 64 bits, w = exp(d); q = ref - logp where there is a reference.
__device__ __forceinline__ PlTerm pl_term(const PlArgs& a, double d, float w, float adv, bool ref, float q) {
    PlTerm r;
    float rise = 0.f;
    r.kl = ref ? pl_kl(q, rise) : 0.f;
    r.kl_slope = a.p.beta != 0.f ? -a.p.beta * rise : 0.f;  // without beta an infinite KL is reported and not added
    const bool below = d < a.log_low, above = d > a.log_high, capped = d > a.log_delta;
    const float weighed = adv == 0.f && d < (double)INFINITY ? 0.f : w * adv;  // exp(d) may overflow where it is finite
    const float first = capped ? a.delta * adv : weighed;
    const float second = below ? a.low * adv : above ? a.high * adv : weighed;
    const float least = second < first ? second : first;  // a NaN of either stays
    r.loss = a.p.beta != 0.f ? fmaf(a.p.beta, r.kl, -least) : -least;
    r.cut_low = below && adv < 0.f;
    r.cut_high = above && adv > 0.f;
    r.slope = (r.cut_low || r.cut_high || capped) ? 0.f : -weighed;
    return r;
}

// What the call returns, from the sums over all tokens.  stats[3]: the factor that the stored gradient still lacks, 1
// where the weight was known before (it is in the gradient then, rounded once with it).
__device__ __forceinline__ void pl_finish(const PlArgs& a, const double* s) {
    const double tokens = s[4] > 1.0 ? s[4] : 1.0;
    const double global = a.constant != 0.0 ? a.constant : 1.0 / tokens;
    a.p.loss[0] = (float)(s[0] * global);
    a.p.stats[0] = (float)(s[1] / tokens);
    a.p.stats[1] = (float)(s[2] / tokens);
    a.p.stats[2] = (float)(s[3] / tokens);
    a.p.stats[3] = a.constant != 0.0 ? 1.f : (float)global;
}

__device__ __forceinline__ void pl_count(PlShare& s, const PlTerm& k) {
    s.loss += (double)k.loss;
    s.kl += (double)k.kl;
    s.low += k.cut_low ? 1 : 0;
    s.high += k.cut_high ? 1 : 0;
    s.valid += 1;
}

// Totals of the workgroup, waves in order; of the only workgroup: the results.
template <int THREADS>
__device__ __forceinline__ void pl_totals(const PlArgs& a, const PlShare& s, double* lds) {
    double sum[PL_SUMS] = {s.total, s.kl, (double)s.low, (double)s.high, (double)s.valid};
#pragma unroll
    for (int i = 0; i < PL_SUMS; ++i) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum[i] += __shfl_xor(sum[i], o, 64);
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < PL_SUMS; ++i) lds[(threadIdx.x >> 6) * PL_SUMS + i] = sum[i];
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 64; ++w)
            for (int i = 0; i < PL_SUMS; ++i) sum[i] += lds[w * PL_SUMS + i];
        if (a.partials == nullptr) {
            pl_finish(a, sum);
        } else {
            for (int i = 0; i < PL_SUMS; ++i) a.partials[(int64_t)blockIdx.x * PL_SUMS + i] = sum[i];
        }
    }
}

// Rows of up to LANES * E tokens, LANES lanes a row, a lane's tokens in registers: every input is read once, and all
// loads of a kind are under way together (masks first, then what they leave).
template <int LANES, int E, int THREADS>
__global__ __launch_bounds__(THREADS) void policy_loss_row_kernel(PlArgs a) {
    __shared__ double lds[16 * PL_SUMS];
    const grx_policy_loss_args& p = a.p;
    constexpr int ROWS = THREADS / LANES;
    const int lane = threadIdx.x % LANES;
    PlShare share = {0.0, 0.0, 0.0, 0, 0, 0};
    for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; r < p.R; r += (int64_t)gridDim.x * ROWS) {
        bool valid[E];
        float x[E], old[E], ref[E], adv[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int t = lane + e * LANES;
            valid[e] = t < p.T && pl_valid(p, r, t);
        }
        const float row_adv = p.adv_pos_stride == 0 ? p.advantages[r * p.adv_row_stride] : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int t = lane + e * LANES;
            x[e] = old[e] = ref[e] = 0.f;
            adv[e] = row_adv;
            if (valid[e]) {
                x[e] = p.logps[r * p.logps_stride + t];
                if (p.old_logps) old[e] = p.old_logps[r * p.old_stride + t];
                if (p.ref_logps) ref[e] = p.ref_logps[r * p.ref_stride + t];
                if (p.adv_pos_stride != 0) adv[e] = p.advantages[r * p.adv_row_stride + (int64_t)t * p.adv_pos_stride];
            }
        }
        // the log ratio of a valid token; without an old policy 0, also where its log-probability is -inf
        const auto ratio = [&](int e) { return p.old_logps ? (double)x[e] - (double)old[e] : 0.0; };
        double row_w = 1.0, inv_n = 1.0, row_d = 0.0;
        const double known = a.constant != 0.0 ? a.constant : 1.0;
        float seq_w = 1.f;
        if (p.row_mean || p.sequence_level) {
            double n = 0.0, d = 0.0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                n += valid[e] ? 1.0 : 0.0;
                if (valid[e]) d += ratio(e);
            }
            n = pl_row_sum<LANES>(n, lds);
            inv_n = 1.0 / (n > 1.0 ? n : 1.0);
            if (p.row_mean) row_w = inv_n;
            if (p.sequence_level) {
                row_d = pl_row_sum<LANES>(d, lds) * inv_n;
                seq_w = expf((float)row_d);
            }
        }
        double slope = 0.0;
        float* grad = p.unit_grad ? p.unit_grad + r * p.T : nullptr;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (valid[e]) {
                double d = row_d;
                float w = seq_w;
                if (!p.sequence_level) {
                    d = ratio(e);
                    w = expf((float)d);
                }
                const PlTerm k = pl_term(a, d, w, adv[e], p.ref_logps != nullptr, (float)((double)ref[e] - (double)x[e]));
                pl_count(share, k);
                if (p.sequence_level) slope += (double)k.slope;
                x[e] = k.slope;
                old[e] = k.kl_slope;
            }
        }
        share.total += row_w * share.loss;
        share.loss = 0.0;
        if (grad == nullptr) continue;
        if (p.sequence_level) slope = pl_row_sum<LANES>(slope, lds) * inv_n;  // every token carries the row's slope
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int t = lane + e * LANES;
            if (t < p.T)
                grad[t] = valid[e] ? (float)(row_w * known * ((p.sequence_level ? slope : (double)x[e]) + (double)old[e])) : 0.f;
        }
    }
    pl_totals<THREADS>(a, share, lds);
}

// Rows of any length, one workgroup a row, in passes over it.
template <int LANES>
__global__ __launch_bounds__(LANES) void policy_loss_kernel(PlArgs a) {
    __shared__ double lds[16 * PL_SUMS];
    const grx_policy_loss_args& p = a.p;
    const int lane = threadIdx.x;
    PlShare share = {0.0, 0.0, 0.0, 0, 0, 0};
    for (int64_t r = blockIdx.x; r < p.R; r += gridDim.x) {
        const float* lp = p.logps + r * p.logps_stride;
        const float* old = p.old_logps ? p.old_logps + r * p.old_stride : nullptr;
        const float* ref = p.ref_logps ? p.ref_logps + r * p.ref_stride : nullptr;
        float* grad = p.unit_grad ? p.unit_grad + r * p.T : nullptr;
        double row_w = 1.0, row_d = 0.0, inv_n = 1.0;
        const double known = a.constant != 0.0 ? a.constant : 1.0;
        if (p.row_mean || p.sequence_level) {
            double n = 0.0, d = 0.0;
            for (int t = lane; t < p.T; t += LANES)
                if (pl_valid(p, r, t)) {
                    n += 1.0;
                    if (p.sequence_level && old) d += (double)lp[t] - (double)old[t];
                }
            n = pl_row_sum<LANES>(n, lds);
            inv_n = 1.0 / (n > 1.0 ? n : 1.0);
            if (p.sequence_level) row_d = pl_row_sum<LANES>(d, lds) * inv_n;
            if (p.row_mean) row_w = inv_n;
        }
        float seq_w = 1.f;
        double seq_slope = 0.0;
        if (p.sequence_level) seq_w = expf((float)row_d);
        for (int pass = 0; pass < (p.sequence_level && grad ? 2 : 1); ++pass) {
            // second pass (one ratio per sequence): every token of the row carries the row's slope
            if (pass == 1) seq_slope = pl_row_sum<LANES>(seq_slope, lds) * inv_n;
            for (int t = lane; t < p.T; t += LANES) {
                if (!pl_valid(p, r, t)) {
                    if (grad && pass == 0) grad[t] = 0.f;
                    continue;
                }
                const float x = lp[t];
                const float q = ref ? (float)((double)ref[t] - (double)x) : 0.f;
                if (pass == 1) {
                    float rise = 0.f;
                    if (p.beta != 0.f) pl_kl(q, rise);
                    grad[t] = (float)(row_w * known * (seq_slope + (double)(-p.beta * rise)));
                    continue;
                }
                double d = row_d;
                float w = seq_w;
                if (!p.sequence_level) {
                    d = old ? (double)x - (double)old[t] : 0.0;
                    w = expf((float)d);
                }
                const PlTerm k = pl_term(a, d, w, p.advantages[r * p.adv_row_stride + (int64_t)t * p.adv_pos_stride], ref, q);
                pl_count(share, k);
                if (!grad) continue;
                if (p.sequence_level)
                    seq_slope += (double)k.slope;
                else
                    grad[t] = (float)(row_w * known * ((double)k.slope + (double)k.kl_slope));
            }
        }
        share.total += row_w * share.loss;
        share.loss = 0.0;
    }
    pl_totals<LANES>(a, share, lds);
}

__global__ __launch_bounds__(PL_THREADS) void policy_loss_join_kernel(PlArgs a) {
    __shared__ double lds[PL_THREADS / 64][PL_SUMS];
    double sum[PL_SUMS] = {0.0, 0.0, 0.0, 0.0, 0.0};
    for (int j = threadIdx.x; j < a.n_partials; j += PL_THREADS)
#pragma unroll
        for (int i = 0; i < PL_SUMS; ++i) sum[i] += a.partials[(int64_t)j * PL_SUMS + i];
#pragma unroll
    for (int i = 0; i < PL_SUMS; ++i) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum[i] += __shfl_xor(sum[i], o, 64);
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6][i] = sum[i];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < PL_THREADS / 64; ++w)
            for (int i = 0; i < PL_SUMS; ++i) sum[i] += lds[w][i];
        pl_finish(a, sum);
    }
}

// dL/dlogps = unit gradient x the factor that was known only at the end x what came from behind the loss
__global__ __launch_bounds__(PL_THREADS) void policy_loss_grad_kernel(const float* __restrict__ unit,
                                                                      const float* __restrict__ stats,
                                                                      const float* __restrict__ upstream, int64_t n,
                                                                      float* __restrict__ out) {
    const float f = stats[3] * upstream[0];
    for (int64_t i = ((int64_t)blockIdx.x * PL_THREADS + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * PL_THREADS * 4) {
        if (i + 4 <= n) {
            const float4 v = *reinterpret_cast<const float4*>(unit + i);
            float4 w;
            w.x = v.x == 0.f ? 0.f : v.x * f;  // padding keeps its 0 under an infinite or NaN factor
            w.y = v.y == 0.f ? 0.f : v.y * f;
            w.z = v.z == 0.f ? 0.f : v.z * f;
            w.w = v.w == 0.f ? 0.f : v.w * f;
            *reinterpret_cast<float4*>(out + i) = w;
        } else {
            for (int64_t j = i; j < n; ++j) out[j] = unit[j] == 0.f ? 0.f : unit[j] * f;
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------
// Lanes per row; a lane's share of a row of up to 1024 tokens stays in registers (4096 rows of 1001 tokens, one ratio a
// row: 30 us with 256 lanes; 64 lanes with 16 tokens each 45 us, for 174 registers leave two waves on a SIMD).
static int pl_lanes(int T) { return T <= 8 ? 8 : T <= 16 ? 16 : T <= 32 ? 32 : T <= 256 ? 64 : T <= 1024 ? PL_THREADS : PL_BIG; }

static int pl_groups(int R, int T) {
    if ((int64_t)R * T <= PL_SINGLE_TOKENS) return 1;
    const int lanes = pl_lanes(T);
    const int rows = lanes == PL_BIG ? 1 : PL_THREADS / lanes;
    const int64_t g = ((int64_t)R + rows - 1) / rows;
    return g < PL_MAX_WGS ? (int)g : PL_MAX_WGS;
}

extern "C" size_t grx_policy_loss_scratch_bytes(int32_t R, int32_t T) {
    if (R <= 0 || T <= 0) return 0;
    const int g = pl_groups(R, T);
    return g > 1 ? (size_t)g * PL_SUMS * sizeof(double) : 0;
}

extern "C" int grx_policy_loss(const grx_policy_loss_args* args, void* scratch, size_t scratch_bytes, void* stream_) {
    const char* who = "grx_policy_loss";
    GRX_REQUIRE(args != nullptr, GRX_E_INVALID, "%s: null args", who);
    PlArgs a;
    memset(&a, 0, sizeof(a));
    a.p = *args;
    const grx_policy_loss_args& p = a.p;
    GRX_REQUIRE(p.R >= 0 && p.T >= 0, GRX_E_INVALID, "%s: bad shape", who);
    GRX_REQUIRE(p.T <= (1 << 30), GRX_E_UNSUPPORTED, "%s: more than 2^30 positions", who);  // positions are stepped over as int
    GRX_REQUIRE(p.loss != nullptr && p.stats != nullptr, GRX_E_INVALID, "%s: null output", who);
    const bool any = (int64_t)p.R * p.T > 0;
    GRX_REQUIRE(!any || (p.logps != nullptr && p.advantages != nullptr && p.mask != nullptr), GRX_E_INVALID,
                "%s: null input", who);
    GRX_REQUIRE(p.mask_type >= GRX_MASK_U8 && p.mask_type <= GRX_MASK_F32, GRX_E_INVALID, "%s: mask type %d", who, p.mask_type);
    GRX_REQUIRE(p.epsilon_low >= 0.0 && p.epsilon_low < 1.0 && p.epsilon_high >= 0.0 && isfinite(p.epsilon_high), GRX_E_INVALID,
                "%s: epsilon_low must lie in [0, 1) and epsilon_high must not be negative", who);
    GRX_REQUIRE(p.delta == 0.0 || (isfinite(p.delta) && p.delta > 1.0 + p.epsilon_high), GRX_E_INVALID,
                "%s: delta must be 0 (off) or above 1 + epsilon_high", who);
    GRX_REQUIRE(isfinite(p.beta) && (p.beta == 0.f || !any || p.ref_logps != nullptr), GRX_E_INVALID,
                "%s: a KL term needs reference log-probabilities", who);
    GRX_REQUIRE(p.normalizer >= 0.0 && isfinite(p.normalizer), GRX_E_INVALID, "%s: normalizer must not be negative", who);
    GRX_REQUIRE(p.unit_grad == nullptr || ((uintptr_t)p.unit_grad & 15) == 0, GRX_E_INVALID, "%s: misaligned unit_grad", who);
    a.log_low = log1p(-p.epsilon_low);
    a.log_high = log1p(p.epsilon_high);
    a.log_delta = p.delta == 0.0 ? (double)INFINITY : log(p.delta);
    a.delta = (float)p.delta;
    a.low = (float)(1.0 - p.epsilon_low);
    a.high = (float)(1.0 + p.epsilon_high);
    a.constant = p.row_mean ? 1.0 / (double)(p.R > 0 ? p.R : 1) : p.normalizer > 0.0 ? 1.0 / p.normalizer : 0.0;
    if (!any) a.p.R = 0;  // rows without positions: nothing is read, their advantages neither
    hipStream_t stream = (hipStream_t)stream_;
    const int lanes = pl_lanes(p.T);
    const int groups = any ? pl_groups(p.R, p.T) : 1;
    a.n_partials = groups;
    if (groups > 1) {
        const size_t need = grx_policy_loss_scratch_bytes(p.R, p.T);
        GRX_REQUIRE(scratch != nullptr && scratch_bytes >= need && ((uintptr_t)scratch & 7) == 0, GRX_E_WORKSPACE,
                    "%s: scratch of %zu bytes, need %zu", who, scratch_bytes, need);
        a.partials = reinterpret_cast<double*>(scratch);
    }
#define PL_LAUNCH(LANES, E)                                                                                          \
    do {                                                                                                             \
        if (groups == 1) hipLaunchKernelGGL((policy_loss_row_kernel<LANES, E, PL_BIG>), dim3(1), dim3(PL_BIG), 0, stream, a); \
        else hipLaunchKernelGGL((policy_loss_row_kernel<LANES, E, PL_THREADS>), dim3(groups), dim3(PL_THREADS), 0, stream, a); \
    } while (0)
    if (lanes == PL_BIG) hipLaunchKernelGGL((policy_loss_kernel<PL_BIG>), dim3(groups), dim3(PL_BIG), 0, stream, a);
    else if (lanes == 8) PL_LAUNCH(8, 1);
    else if (lanes == 16) PL_LAUNCH(16, 1);
    else if (lanes == 32) PL_LAUNCH(32, 1);
    else if (p.T <= 64) PL_LAUNCH(64, 1);
    else if (p.T <= 256) PL_LAUNCH(64, 4);
    else hipLaunchKernelGGL((policy_loss_row_kernel<PL_THREADS, 4, PL_THREADS>), dim3(groups), dim3(PL_THREADS), 0, stream, a);
    GRX_CHECK_HIP(hipGetLastError());
    if (groups > 1) {
        hipLaunchKernelGGL(policy_loss_join_kernel, dim3(1), dim3(PL_THREADS), 0, stream, a);
        GRX_CHECK_HIP(hipGetLastError());
    }
    return GRX_OK;
}

extern "C" int grx_policy_loss_backward(const float* unit_grad, const float* stats, const float* upstream, int64_t n,
                                        float* grad_logps, void* stream_) {
    const char* who = "grx_policy_loss_backward";
    GRX_REQUIRE(n >= 0, GRX_E_INVALID, "%s: bad size", who);
    if (n == 0) return GRX_OK;
    GRX_REQUIRE(unit_grad != nullptr && stats != nullptr && upstream != nullptr && grad_logps != nullptr, GRX_E_INVALID,
                "%s: null buffer", who);
    GRX_REQUIRE((((uintptr_t)unit_grad | (uintptr_t)grad_logps) & 15) == 0, GRX_E_INVALID, "%s: misaligned buffer", who);
    int64_t wgs = (n / 4 + PL_THREADS - 1) / PL_THREADS;
    wgs = wgs < 1 ? 1 : wgs > 2048 ? 2048 : wgs;
    hipLaunchKernelGGL(policy_loss_grad_kernel, dim3((unsigned)wgs), dim3(PL_THREADS), 0, (hipStream_t)stream_, unit_grad,
                       stats, upstream, n, grad_logps);
    GRX_CHECK_HIP(hipGetLastError());
    return GRX_OK;
}

extern "C" size_t grx_policy_struct_bytes(int32_t which) {
    return which == 0 ? sizeof(grx_token_logps_args) : which == 1 ? sizeof(grx_lm_token_logps_args) : which == 2 ? sizeof(grx_policy_loss_args) : 0;
}
