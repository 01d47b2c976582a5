// Log-probabilities and entropies of chosen tokens from logits, and the gradient of the logits: what a
// policy-gradient step needs of the policy's output.  Per row of V logits x, with T the temperature,
//   lse = log sum_v exp(x_v / T),   logp = x_t / T - lse,   H = lse - sum_v p_v x_v / T,   p_v = exp(x_v / T - lse),
//   dL/dx_v = (g [v == t] - p_v (g + h (log p_v + H))) / T     for dL/dlogp = g, dL/dH = h.
// Both directions are one pass over the rows and bound by HBM: about ten lane operations per element, and the
// row's (max, sum of exponentials) is all that the backward pass needs besides the logits.  Rows whose token id
// is negative are padding: they are not read, and have log-probability, entropy and gradient 0.
// The rows are larger than the caches between one pass and the next, so loads and stores are non-temporal: 8192 rows
// of 152,640 bf16 forward 363 us (6.9 TB/s, what a plain read of them reaches), with ordinary ones 449 us.
#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>

#include "common.h"
#include "lse_math.h"

#define TL_THREADS 256
#define TL_WAVES (TL_THREADS / GRX_WAVE)
#define TL_WIDE 1024
#define TL_UNROLL 4          // 16-byte loads in flight per thread
#define TL_MAX_PARTS 64
// Rows are split until there are this many workgroups (eight of them run on a CU): 1280 rows, 41 % of them padding, take
// 49 us split three ways and 54 us whole, 1073 fp32 rows 64 and 100 us; 16,384 workgroups are no better than 4096.
#define TL_TARGET_WGS 4096
#define TL_FLOOR (-200.f)    // 2^-200 is 0 in fp32: keeps 0 * -inf out of the entropy sums

typedef u32x4 u32x4_any __attribute__((aligned(2)));  // rows start at any element

struct TlArgs {
    const void* logits;
    int64_t stride_b, stride_t;
    const int64_t* ids;
    int64_t ids_stride;
    int T, V;
    float k;                 // log2(e) / temperature
    float inv_t;
    int parts;
    float* logps;
    float2* stats;
    float* entropy;
    float4* partials;        // [rows][parts] (max, sum, weighted sum), parts > 1
    const float* g;
    const float* h;
    void* grad;
    int n_chunks;
    int row0;                // first row of the launch
};

// A thread's share: m = largest logit, s = sum of 2^((x - m) k), u = sum of the same times (x - m) k.
// The difference is taken before the factor: rows of any finite logits, the type's lowest value among them,
// stay finite.  A NaN among the logits is dropped by the maximum and kept by the sum.
struct Share {
    float m, s, u;
};

template <bool ENT>
__device__ __forceinline__ Share share_merge(const Share& a, const Share& b, float k) {
    Share r;
    r.m = fmaxf(a.m, b.m);
    const float ref = r.m == -INFINITY ? 0.f : r.m;
    const float da = fmaxf((a.m - ref) * k, TL_FLOOR), db = fmaxf((b.m - ref) * k, TL_FLOOR);
    const float fa = fast_exp2(da), fb = fast_exp2(db);
    r.s = a.s * fa + b.s * fb;
    r.u = ENT ? (a.u + a.s * da) * fa + (b.u + b.s * db) * fb : 0.f;
    return r;
}

template <bool ENT, int N>
__device__ __forceinline__ void share_add(Share& a, const float* x, float k) {
    float m = a.m;
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, x[j]);
    const float ref = m == -INFINITY ? 0.f : m;
    const float d = fmaxf((a.m - ref) * k, TL_FLOOR);
    const float f = fast_exp2(d);
    float s0 = 0.f, s1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float t = (x[j] - ref) * k;
        const float w = fast_exp2(t);
        if (j & 1) s1 += w; else s0 += w;
        if (ENT) {
            const float tc = fmaxf(t, TL_FLOOR);
            if (j & 1) u1 = fmaf(w, tc, u1); else u0 = fmaf(w, tc, u0);
        }
    }
    if (ENT) a.u = (a.u + a.s * d) * f + (u0 + u1);
    a.s = a.s * f + (s0 + s1);
    a.m = m;
}

template <bool ENT, int THREADS>
__device__ __forceinline__ Share share_block(Share a, float k, Share* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        Share b;
        b.m = __shfl_xor(a.m, o, GRX_WAVE);
        b.s = __shfl_xor(a.s, o, GRX_WAVE);
        b.u = ENT ? __shfl_xor(a.u, o, GRX_WAVE) : 0.f;
        a = share_merge<ENT>(a, b, k);
    }
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    a = lds[0];
#pragma unroll
    for (int w = 1; w < THREADS / GRX_WAVE; ++w) a = share_merge<ENT>(a, lds[w], k);
    return a;
}

template <int DT>
__device__ __forceinline__ const typename Elem<DT>::T* tl_row(const TlArgs& a, int row) {
    const int b = row / a.T, t = row - b * a.T;
    return reinterpret_cast<const typename Elem<DT>::T*>(a.logits) + (int64_t)b * a.stride_b + (int64_t)t * a.stride_t;
}

__device__ __forceinline__ int64_t tl_id(const TlArgs& a, int row) {
    const int b = row / a.T, t = row - b * a.T;
    return a.ids[(int64_t)b * a.ids_stride + t];
}

// Row results from its complete sums.  A token id outside the vocabulary has no log-probability: NaN.
template <int DT>
__device__ __forceinline__ void tl_finish(const TlArgs& a, int row, int64_t id, const Share& sh) {
    const float ls = log2f(sh.s);
    const float ln2 = 0.69314718055994531f;
    float lp = NAN;
    if (id < a.V) lp = ((Elem<DT>::to_float(tl_row<DT>(a, row)[id]) - sh.m) * a.k - ls) * ln2;
    a.logps[row] = lp;
    a.stats[row] = make_float2(sh.m, sh.s);
    if (a.entropy) a.entropy[row] = (ls - sh.u / sh.s) * ln2;
}

__device__ __forceinline__ void tl_finish_padding(const TlArgs& a, int row) {
    a.logps[row] = 0.f;
    a.stats[row] = make_float2(0.f, 1.f);
    if (a.entropy) a.entropy[row] = 0.f;
}

template <int DT, bool ENT, int THREADS>
__device__ __forceinline__ void tl_forward(const TlArgs& a) {
    typedef typename Elem<DT>::T T;
    constexpr int PV = Elem<DT>::kPerVec;
    __shared__ Share lds[THREADS / GRX_WAVE];
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const int64_t id = tl_id(a, row);
    if (id < 0) {
        if (a.parts == 1 && threadIdx.x == 0) tl_finish_padding(a, row);
        return;
    }
    const T* __restrict__ x = tl_row<DT>(a, row);
    // elements before the first 16-byte boundary, whole vectors, elements behind the last one
    int head = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T));
    if (head > a.V) head = a.V;
    const int n_vec = (a.V - head) / PV;
    const int per = (n_vec + a.parts - 1) / a.parts;
    const int v0 = part * per < n_vec ? part * per : n_vec;
    const int v1 = v0 + per < n_vec ? v0 + per : n_vec;
    Share sh = {-INFINITY, 0.f, 0.f};
    const u32x4* __restrict__ body = reinterpret_cast<const u32x4*>(x + head);
    int i = v0 + threadIdx.x;
    for (; i + (TL_UNROLL - 1) * THREADS < v1; i += TL_UNROLL * THREADS) {
        u32x4 q[TL_UNROLL];
#pragma unroll
        for (int j = 0; j < TL_UNROLL; ++j) q[j] = __builtin_nontemporal_load(body + i + j * THREADS);
        float f[TL_UNROLL * PV];
#pragma unroll
        for (int j = 0; j < TL_UNROLL; ++j) Elem<DT>::unpack(q[j], f + j * PV);
        share_add<ENT, TL_UNROLL * PV>(sh, f, a.k);
    }
    for (; i < v1; i += THREADS) {
        float f[PV];
        Elem<DT>::unpack(body[i], f);
        share_add<ENT, PV>(sh, f, a.k);
    }
    if (part == 0 && (int)threadIdx.x < head) {
        const float f = Elem<DT>::to_float(x[threadIdx.x]);
        share_add<ENT, 1>(sh, &f, a.k);
    }
    const int tail = head + n_vec * PV + threadIdx.x;
    if (part == a.parts - 1 && tail < a.V) {
        const float f = Elem<DT>::to_float(x[tail]);
        share_add<ENT, 1>(sh, &f, a.k);
    }
    sh = share_block<ENT, THREADS>(sh, a.k, lds);
    if (threadIdx.x == 0) {
        if (a.parts == 1)
            tl_finish<DT>(a, row, id, sh);
        else
            a.partials[(int64_t)row * a.parts + part] = make_float4(sh.m, sh.s, sh.u, 0.f);
    }
}

template <int DT, bool ENT>
__global__ __launch_bounds__(TL_THREADS) void token_logps_kernel(TlArgs a) {
    tl_forward<DT, ENT, TL_THREADS>(a);
}

template <int DT, bool ENT>
__global__ __launch_bounds__(TL_WIDE) void token_logps_wide_kernel(TlArgs a) {
    tl_forward<DT, ENT, TL_WIDE>(a);
}

// Joins the parts of split rows, one wave per row (at most TL_MAX_PARTS = 64 parts).
template <int DT, bool ENT>
__global__ __launch_bounds__(TL_THREADS) void token_logps_join_kernel(TlArgs a, int rows) {
    const int row = blockIdx.x * TL_WAVES + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= rows) return;
    const int64_t id = tl_id(a, row);
    if (id < 0) {
        if (lane == 0) tl_finish_padding(a, row);
        return;
    }
    Share sh = {-INFINITY, 0.f, 0.f};
    if (lane < a.parts) {
        const float4 p = a.partials[(int64_t)row * a.parts + lane];
        sh = {p.x, p.y, p.z};
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        Share b;
        b.m = __shfl_xor(sh.m, o, GRX_WAVE);
        b.s = __shfl_xor(sh.s, o, GRX_WAVE);
        b.u = __shfl_xor(sh.u, o, GRX_WAVE);
        sh = share_merge<ENT>(sh, b, a.k);
    }
    if (lane == 0) tl_finish<DT>(a, row, id, sh);
}

template <int DT>
__device__ __forceinline__ u32x4 tl_pack(const float* f);
template <>
__device__ __forceinline__ u32x4 tl_pack<GRX_F32>(const float* f) {
    return u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
}
template <>
__device__ __forceinline__ u32x4 tl_pack<GRX_BF16>(const float* f) {
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
    const f32x8 v = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
    return __builtin_bit_cast(u32x4, __builtin_convertvector(v, b16x8));
}
template <>
__device__ __forceinline__ u32x4 tl_pack<GRX_F16>(const float* f) {
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
    const f32x8 v = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
    return __builtin_bit_cast(u32x4, __builtin_convertvector(v, h16x8));
}

// 8 KB of gradient per workgroup: two loads a thread.  8192 rows of 152,640 bf16: 780 us (6.4 TB/s), with 4, 16 and
// 32 KB 950, 837 and 905 us.
#define TL_CHUNK_VECS (TL_THREADS * 2)

// Gradient: w = 2^((x - m) k), dx = w (alpha + beta t) with t = (x - m) k, plus g / T at the token.
template <int DT, bool ENT>
__global__ __launch_bounds__(TL_THREADS) void token_logps_grad_kernel(TlArgs a) {
    typedef typename Elem<DT>::T T;
    constexpr int PV = Elem<DT>::kPerVec;
    const int at_row = blockIdx.x / a.n_chunks, chunk = blockIdx.x - at_row * a.n_chunks, row = a.row0 + at_row;
    const int64_t id = tl_id(a, row);
    T* __restrict__ d = reinterpret_cast<T*>(a.grad) + (int64_t)row * a.V;
    int head = (int)(((16 - ((uintptr_t)d & 15)) & 15) / sizeof(T));
    if (head > a.V) head = a.V;
    const int n_vec = (a.V - head) / PV;
    const int v0 = chunk * TL_CHUNK_VECS, v1 = v0 + TL_CHUNK_VECS < n_vec ? v0 + TL_CHUNK_VECS : n_vec;
    u32x4* __restrict__ dv = reinterpret_cast<u32x4*>(d + head);
    const int edge = chunk == 0 && (int)threadIdx.x < head ? (int)threadIdx.x : -1;
    int last = head + n_vec * PV + threadIdx.x;
    if (chunk != a.n_chunks - 1 || last >= a.V) last = -1;
    const float g = id < 0 ? 0.f : a.g ? a.g[row] : 0.f;
    const float h = ENT && id >= 0 && a.h ? a.h[row] : 0.f;
    if (g == 0.f && h == 0.f) {  // padding, or a token that the loss left out: nothing to read
        for (int i = v0 + threadIdx.x; i < v1; i += TL_THREADS) dv[i] = u32x4{0, 0, 0, 0};
        if (edge >= 0) d[edge] = (T)0;
        if (last >= 0) d[last] = (T)0;
        return;
    }
    const T* __restrict__ x = tl_row<DT>(a, row);
    const float2 st = a.stats[row];
    const float m = st.x, k = a.k;
    float alpha, beta = 0.f;
    if (ENT) {
        const float ln2 = 0.69314718055994531f;
        alpha = -(g + h * (a.entropy[row] - log2f(st.y) * ln2)) * a.inv_t / st.y;
        beta = -h * ln2 * a.inv_t / st.y;
    } else {
        alpha = -g * a.inv_t / st.y;
    }
    const float at = id < a.V ? g * a.inv_t : NAN;
    const int tok = id < a.V ? (int)id : 0;
    auto one = [&](float xv) {
        const float t = (xv - m) * k;
        const float w = fast_exp2(t);
        return ENT ? w * fmaf(beta, fmaxf(t, TL_FLOOR), alpha) : w * alpha;
    };
    const u32x4_any* __restrict__ xv = reinterpret_cast<const u32x4_any*>(x + head);
    for (int i = v0 + threadIdx.x; i < v1; i += TL_THREADS) {
        float f[PV];
        const u32x4 q = __builtin_nontemporal_load(xv + i);
        Elem<DT>::unpack(q, f);
#pragma unroll
        for (int j = 0; j < PV; ++j) f[j] = one(f[j]);
        const int e = tok - (head + i * PV);
        if ((unsigned)e < (unsigned)PV) {
#pragma unroll
            for (int j = 0; j < PV; ++j)
                if (j == e) f[j] += at;
        }
        __builtin_nontemporal_store(tl_pack<DT>(f), dv + i);
    }
    if (edge >= 0) d[edge] = Elem<DT>::from_float(one(Elem<DT>::to_float(x[edge])) + (edge == tok ? at : 0.f));
    if (last >= 0) d[last] = Elem<DT>::from_float(one(Elem<DT>::to_float(x[last])) + (last == tok ? at : 0.f));
}

// ---- host ------------------------------------------------------------------------------------------
// Rows that fill the CUs once, or twice to three quarters and more (a CU holds two workgroups of 1024 threads), and are
// long enough for a turn of the loop: whole, in one launch.  Kernel times in us, whole and split:
//   rows                             112          160          256          320          384          512
//   V = 152,640 bf16           13.3 12.0    14.0 14.8    16.1 19.5    24.5 24.4    25.5 27.7    29.2 32.3
//     with entropies           15.2 12.9    16.0 16.0    17.7 21.4    27.3 26.7    27.8 30.2    30.9 34.8
//     40 % of them padding     12.9 11.4    13.1 12.7    13.5 14.9    21.4 17.4    21.8 19.5    23.2 23.7
//   V = 152,640 fp32           16.3 14.6    19.8 22.1    26.3 28.7    37.7 35.9    41.1 41.6    50.3 54.8
//   V =  33,000 bf16            6.6  7.7     6.7  8.0     7.0  9.2     9.6  9.8     9.6 10.8     9.9 12.1
//   V =  80,000 fp32, entropies 11.0 11.5   12.7 13.8    15.1 21.0    22.2 24.9    23.6 28.5    28.2 31.3
// With padding workgroups that find nothing to do cost a part of what is won, and with more rows all of it (1280 rows, half of
// them padding: 52 and 49).
static bool tl_wide(int64_t rows, int V, int dtype) {
    const int64_t bytes = (int64_t)V * (dtype == GRX_F32 ? 4 : 2);
    return rows >= 128 && rows <= 512 && (rows <= 256 || rows >= 384) && bytes >= TL_WIDE * TL_UNROLL * 16;
}

static int tl_parts(int64_t rows, int V, int dtype) {
    if (tl_wide(rows, V, dtype)) return 1;
    const int64_t vecs = ((int64_t)V * (dtype == GRX_F32 ? 4 : 2) + 15) / 16;
    int64_t p = rows > 0 ? (TL_TARGET_WGS + rows - 1) / rows : 1;
    // at least one turn of the loop per part; of few rows, at least one load per thread
    const int64_t most = vecs / (rows < 64 ? TL_THREADS : TL_THREADS * TL_UNROLL);
    if (p > most) p = most;
    if (p > TL_MAX_PARTS) p = TL_MAX_PARTS;
    return p < 2 ? 1 : (int)p;
}

extern "C" size_t grx_token_logps_scratch_bytes(int64_t rows, int32_t V, int32_t dtype) {
    if (rows <= 0 || V <= 0) return 0;
    const int p = tl_parts(rows, V, dtype);
    return p > 1 ? (size_t)rows * (size_t)p * sizeof(float4) : 0;
}

static int tl_check(const char* who, const grx_token_logps_args* p) {
    GRX_REQUIRE(p != nullptr, GRX_E_INVALID, "%s: null args", who);
    GRX_REQUIRE(p->B >= 0 && p->T >= 0 && p->V >= 1, GRX_E_INVALID, "%s: bad shape", who);
    GRX_REQUIRE(p->dtype == GRX_F32 || p->dtype == GRX_BF16 || p->dtype == GRX_F16, GRX_E_UNSUPPORTED, "%s: dtype %d", who,
                p->dtype);
    GRX_REQUIRE((int64_t)p->B * p->T <= GRX_MAX_TOKEN_ROWS, GRX_E_UNSUPPORTED, "%s: more than %d rows", who,
                GRX_MAX_TOKEN_ROWS);
    GRX_REQUIRE(p->V <= (1 << 24), GRX_E_UNSUPPORTED, "%s: vocabulary above 2^24", who);
    // its inverse has to be finite too
    GRX_REQUIRE(p->temperature >= FLT_MIN && p->temperature < INFINITY, GRX_E_INVALID, "%s: temperature must be at least 2^-126", who);
    if ((int64_t)p->B * p->T == 0) return GRX_OK;
    GRX_REQUIRE(p->logits != nullptr && p->token_ids != nullptr && p->row_stats != nullptr, GRX_E_INVALID,
                "%s: null buffer", who);
    const uintptr_t size = p->dtype == GRX_F32 ? 4 : 2;
    GRX_REQUIRE(((uintptr_t)p->logits % size) == 0 && ((uintptr_t)p->row_stats & 7) == 0, GRX_E_INVALID,
                "%s: misaligned buffer", who);
    return GRX_OK;
}

static TlArgs tl_args(const grx_token_logps_args* p) {
    TlArgs a;
    a.logits = p->logits;
    a.stride_b = p->row_stride;
    a.stride_t = p->pos_stride;
    a.ids = p->token_ids;
    a.ids_stride = p->ids_stride;
    a.T = p->T;
    a.V = p->V;
    a.k = (float)(1.4426950408889634 / (double)p->temperature);
    a.inv_t = (float)(1.0 / (double)p->temperature);
    a.parts = 1;
    a.logps = p->logps;
    a.stats = reinterpret_cast<float2*>(p->row_stats);
    a.entropy = p->entropy;
    a.partials = nullptr;
    a.g = p->grad_logps;
    a.h = p->grad_entropy;
    a.grad = p->grad_logits;
    a.n_chunks = 1;
    a.row0 = 0;
    return a;
}

#define TL_LAUNCH(kernel, grid, threads, ...)                                                                     \
    do {                                                                                                          \
        const dim3 g_((unsigned)(grid)), b_(threads);                                                             \
        if (p->dtype == GRX_F32) {                                                                                \
            if (ent) hipLaunchKernelGGL((kernel<GRX_F32, true>), g_, b_, 0, stream, __VA_ARGS__);                  \
            else hipLaunchKernelGGL((kernel<GRX_F32, false>), g_, b_, 0, stream, __VA_ARGS__);                     \
        } else if (p->dtype == GRX_BF16) {                                                                        \
            if (ent) hipLaunchKernelGGL((kernel<GRX_BF16, true>), g_, b_, 0, stream, __VA_ARGS__);                 \
            else hipLaunchKernelGGL((kernel<GRX_BF16, false>), g_, b_, 0, stream, __VA_ARGS__);                    \
        } else {                                                                                                  \
            if (ent) hipLaunchKernelGGL((kernel<GRX_F16, true>), g_, b_, 0, stream, __VA_ARGS__);                  \
            else hipLaunchKernelGGL((kernel<GRX_F16, false>), g_, b_, 0, stream, __VA_ARGS__);                     \
        }                                                                                                         \
        GRX_CHECK_HIP(hipGetLastError());                                                                         \
    } while (0)

extern "C" int grx_token_logps(const grx_token_logps_args* p, void* scratch, size_t scratch_bytes, void* stream_) {
    const char* who = "grx_token_logps";
    const int rc = tl_check(who, p);
    if (rc != GRX_OK) return rc;
    const int64_t rows = (int64_t)p->B * p->T;
    if (rows == 0) return GRX_OK;
    GRX_REQUIRE(p->logps != nullptr, GRX_E_INVALID, "%s: null logps", who);
    hipStream_t stream = (hipStream_t)stream_;
    const bool ent = p->entropy != nullptr;
    TlArgs a = tl_args(p);
    a.parts = tl_parts(rows, p->V, p->dtype);
    if (a.parts > 1) {
        const size_t need = grx_token_logps_scratch_bytes(rows, p->V, p->dtype);
        GRX_REQUIRE(scratch != nullptr && scratch_bytes >= need, GRX_E_WORKSPACE, "%s: scratch of %zu bytes, need %zu", who,
                    scratch_bytes, need);
        GRX_REQUIRE(((uintptr_t)scratch & 15) == 0, GRX_E_INVALID, "%s: misaligned scratch", who);
        a.partials = reinterpret_cast<float4*>(scratch);
    }
    if (tl_wide(rows, p->V, p->dtype)) {
        TL_LAUNCH(token_logps_wide_kernel, rows, TL_WIDE, a);
        return GRX_OK;
    }
    TL_LAUNCH(token_logps_kernel, rows * a.parts, TL_THREADS, a);
    if (a.parts > 1) TL_LAUNCH(token_logps_join_kernel, (rows + TL_WAVES - 1) / TL_WAVES, TL_THREADS, a, (int)rows);
    return GRX_OK;
}

extern "C" int grx_token_logps_backward(const grx_token_logps_args* p, void* stream_) {
    const char* who = "grx_token_logps_backward";
    const int rc = tl_check(who, p);
    if (rc != GRX_OK) return rc;
    const int64_t rows = (int64_t)p->B * p->T;
    if (rows == 0) return GRX_OK;
    GRX_REQUIRE(p->grad_logits != nullptr, GRX_E_INVALID, "%s: null grad_logits", who);
    GRX_REQUIRE(((uintptr_t)p->grad_logits % (p->dtype == GRX_F32 ? 4 : 2)) == 0, GRX_E_INVALID, "%s: misaligned grad_logits",
                who);
    GRX_REQUIRE(p->grad_entropy == nullptr || p->entropy != nullptr, GRX_E_INVALID,
                "%s: a gradient of the entropies needs the entropies", who);
    hipStream_t stream = (hipStream_t)stream_;
    const bool ent = p->grad_entropy != nullptr;
    TlArgs a = tl_args(p);
    const int pv = p->dtype == GRX_F32 ? 4 : 8;
    a.n_chunks = (p->V / pv + TL_CHUNK_VECS - 1) / TL_CHUNK_VECS;
    if (a.n_chunks < 1) a.n_chunks = 1;
    const int64_t most = ((1 << 24) - 1) / a.n_chunks;  // a launch holds fewer than 2^32 threads
    for (int64_t row = 0; row < rows; row += most) {
        a.row0 = (int)row;
        TL_LAUNCH(token_logps_grad_kernel, (rows - row < most ? rows - row : most) * a.n_chunks, TL_THREADS, a);
    }
    return GRX_OK;
}
