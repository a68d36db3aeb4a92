// Causal depth-wise convolution over time, the short one in front of a selective scan, channels-last:
//   pre[b][t][d] = bias[d] + sum_{k < K} w[d][k] x[b][t - K + 1 + k][d],   y = silu(pre) or pre,   K <= 8,
// with the K - 1 inputs before token 0 taken from `state` [B][K-1][D] (zeros without one), a length per row of a padded batch, and the K - 1 inputs before
// each row's end returned as the state that the next call or the single-token form takes.
// Bound: HBM.  A thread owns V neighbouring channels (16 bytes where alignment allows) and walks a run of tokens with the window in registers, so every
// input is loaded once per run plus K - 1 of the run before it; four tokens are asked for at a time.  All arithmetic is fp32; x, y, state and their gradients
// are rounded once, on the way out.
// 32768 tokens of 2304 channels, bf16 (302 MB): 65 us, 4.6 TB/s.  2048 rows of 125 tokens, 192 channels, fp32: 71 us (393 MB), gradients 161 us (590 MB, 3.7 TB/s).
#include "common.h"

namespace rtfs {

typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));

// V values as they are loaded (16 bytes, or one)
template <typename T, int V> struct ConvRaw;
template <> struct ConvRaw<float, 1> { float v; };
template <> struct ConvRaw<__bf16, 1> { __bf16 v; };
template <> struct ConvRaw<float, 4> { float4 v; };
template <> struct ConvRaw<__bf16, 8> { bhalf8 v; };

template <typename T, int V>
__device__ __forceinline__ ConvRaw<T, V> conv_raw(const T* p) { return *reinterpret_cast<const ConvRaw<T, V>*>(p); }
template <typename T, int V>
__device__ __forceinline__ void conv_widen(const ConvRaw<T, V>& a, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = (float)a.v;
    } else if constexpr (sizeof(T) == 4) {
        v[0] = a.v.x, v[1] = a.v.y, v[2] = a.v.z, v[3] = a.v.w;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)a.v[e];
    }
}
template <typename T, int V>
__device__ __forceinline__ void conv_load(const T* p, float (&v)[V]) { conv_widen<T, V>(conv_raw<T, V>(p), v); }
template <typename T, int V>
__device__ __forceinline__ void conv_store(T* p, const float (&v)[V]) {
    if constexpr (V == 1) {
        *p = (T)v[0];
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        bhalf8 a;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = (__bf16)v[e];
        *reinterpret_cast<bhalf8*>(p) = a;
    }
}
template <int V>
__device__ __forceinline__ void conv_zero(float (&v)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
}

struct ConvArgs {
    const void* x;
    long long x_row, x_tok;  // elements from row to row and from token to token
    const float *w, *bias;
    const void* state;
    const int* lengths;
    int B, L, D, silu;
    int tile_log2, tiles;  // channel vectors per workgroup row (a power of two), workgroup rows across D
    int run, runs;         // tokens per thread, runs per row of the batch
};

__device__ __forceinline__ int conv_length(const ConvArgs& a, int b) {
    if (!a.lengths) return a.L;
    const int n = a.lengths[b];
    return n < 0 ? 0 : n < a.L ? n : a.L;
}
// input of row b at token t >= -(K-1), t < the row's length
template <typename T, int K, int V>
__device__ __forceinline__ void conv_input(const ConvArgs& a, int b, int t, int d, float (&v)[V]) {
    if (t >= 0) conv_load<T, V>(static_cast<const T*>(a.x) + b * a.x_row + t * a.x_tok + d, v);
    else if (a.state) conv_load<T, V>(static_cast<const T*>(a.state) + ((long long)b * (K - 1) + t + K - 1) * a.D + d, v);
    else conv_zero(v);
}
template <int K, int V>
__device__ __forceinline__ void conv_weights(const ConvArgs& a, int d, float (&w)[K][V], float (&bias)[V]) {
    float all[V][K];
    const float* from = a.w + (long long)d * K;
    if constexpr (V == 1) {
#pragma unroll
        for (int k = 0; k < K; ++k) all[0][k] = from[k];
        bias[0] = a.bias ? a.bias[d] : 0.f;
    } else {  // the weights of V neighbouring channels are V K neighbouring values
#pragma unroll
        for (int i = 0; i < V * K; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(from + i);
            all[i / K][i % K] = v.x, all[(i + 1) / K][(i + 1) % K] = v.y, all[(i + 2) / K][(i + 2) % K] = v.z, all[(i + 3) / K][(i + 3) % K] = v.w;
        }
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float4 v = a.bias ? *reinterpret_cast<const float4*>(a.bias + d + e) : make_float4(0.f, 0.f, 0.f, 0.f);
            bias[e] = v.x, bias[e + 1] = v.y, bias[e + 2] = v.z, bias[e + 3] = v.w;
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) w[k][e] = all[e][k];
}

constexpr int kConvAhead = 4;  // tokens asked for at a time

template <typename T, int K, int V>
__global__ __launch_bounds__(256) void causal_conv_kernel(ConvArgs a, T* __restrict__ y, T* __restrict__ last) {
    const int tile = blockIdx.x % a.tiles, across = 1 << a.tile_log2;
    const int d = ((tile << a.tile_log2) + (threadIdx.x & (across - 1))) * V;
    const long long which = (long long)(blockIdx.x / a.tiles) * (256 >> a.tile_log2) + (threadIdx.x >> a.tile_log2);
    if (d >= a.D || which >= (long long)a.B * a.runs) return;
    const int b = (int)(which / a.runs), t0 = (int)(which % a.runs) * a.run;
    const int len = conv_length(a, b), t1 = t0 + a.run < a.L ? t0 + a.run : a.L;
    float w[K][V], bias[V], win[K][V];
    conv_weights<K, V>(a, d, w, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        if (t0 - (K - 1) + k < len) conv_input<T, K, V>(a, b, t0 - (K - 1) + k, d, win[k + 1]);
        else conv_zero(win[k + 1]);
    }
    T* out = y + ((long long)b * a.L + t0) * a.D + d;
    const T* in = static_cast<const T*>(a.x) + b * a.x_row + d;
    const int end = len > 0 ? len - 1 : 0;  // loads go no further: a token behind the row's end counts as zero whatever is read in its place
    for (int tb = t0; tb < t1; tb += kConvAhead) {
        ConvRaw<T, V> raw[kConvAhead];
#pragma unroll
        for (int i = 0; i < kConvAhead; ++i) raw[i] = conv_raw<T, V>(in + (long long)(tb + i < end ? tb + i : end) * a.x_tok);
#pragma unroll
        for (int i = 0; i < kConvAhead; ++i, out += a.D) {
            float o[V];
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) win[k][e] = win[k + 1][e];
            conv_widen<T, V>(raw[i], win[K - 1]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float s = bias[e];
#pragma unroll
                for (int k = 0; k < K; ++k) s = fmaf(w[k][e], win[k][e], s);
                o[e] = tb + i >= len ? 0.f : a.silu ? s * sigmoidf_fast(s) : s;
            }
            if (tb + i < t1) conv_store<T, V>(out, o);
        }
    }
    if (last && t0 == 0) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            float v[V];
            conv_input<T, K, V>(a, b, len - (K - 1) + j, d, v);
            conv_store<T, V>(last + ((long long)b * (K - 1) + j) * a.D + d, v);
        }
    }
}

// Adjoint.  A thread walks its run forwards with two windows, the inputs and dpre = dy silu'(pre) (pre is formed again: cheaper than a stored one), and
// K - 1 tokens past its end for the dpre that reach back into the run:  dx[u] = sum_k w[k] dpre[u + K - 1 - k].  The first run of a row emits the state's
// gradient as the tokens -(K-1) .. -1.  dw[k] = sum_t dpre[t] x[t - K + 1 + k] and dbias are kept in registers over all runs that a workgroup takes, joined
// in LDS and left as ONE partial row per workgroup, which conv_finish_kernel adds in order: the same bits on every run.
template <typename T, int K, int V>
__global__ __launch_bounds__(256) void causal_conv_bwd_kernel(ConvArgs a, const T* __restrict__ dy, const T* __restrict__ dlast, T* __restrict__ dx,
                                                              T* __restrict__ dstate, float* __restrict__ parts) {
    __shared__ float red[256 * V];
    const int tile = blockIdx.x % a.tiles, group = blockIdx.x / a.tiles, groups = gridDim.x / a.tiles, across = 1 << a.tile_log2;
    const int d = ((tile << a.tile_log2) + (threadIdx.x & (across - 1))) * V;
    const bool inside = d < a.D;
    float w[K][V], bias[V], dw[K + 1][V];
    if (inside) conv_weights<K, V>(a, d, w, bias);
#pragma unroll
    for (int k = 0; k <= K; ++k) conv_zero(dw[k]);
    const long long step = 256 >> a.tile_log2;
    for (long long which = (long long)group * step + (threadIdx.x >> a.tile_log2); inside && which < (long long)a.B * a.runs; which += groups * step) {
        const int b = (int)(which / a.runs), t0 = (int)(which % a.runs) * a.run;
        const int len = conv_length(a, b), t1 = t0 + a.run < a.L ? t0 + a.run : a.L;
        float win[K][V], g[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k) conv_zero(g[k]);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            if (t0 - (K - 1) + k < len) conv_input<T, K, V>(a, b, t0 - (K - 1) + k, d, win[k + 1]);
            else conv_zero(win[k + 1]);
        }
        const T* in = static_cast<const T*>(a.x) + b * a.x_row + d;
        const T* din = dy + (long long)b * a.L * a.D + d;
        const int end = len > 0 ? len - 1 : 0;
        for (int tb = t0; tb < t1 + K - 1; tb += kConvAhead) {
            ConvRaw<T, V> rx[kConvAhead], rg[kConvAhead];
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) {
                const int t = tb + i < end ? tb + i : end;
                rx[i] = conv_raw<T, V>(in + (long long)t * a.x_tok);
                rg[i] = conv_raw<T, V>(din + (long long)t * a.D);
            }
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) {
                const int t = tb + i;
                if (t >= t1 + K - 1) break;
#pragma unroll
                for (int k = 0; k < K - 1; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) win[k][e] = win[k + 1][e], g[k][e] = g[k + 1][e];
                conv_widen<T, V>(rx[i], win[K - 1]);
                conv_widen<T, V>(rg[i], g[K - 1]);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (a.silu) {
                        float s = bias[e];
#pragma unroll
                        for (int k = 0; k < K; ++k) s = fmaf(w[k][e], win[k][e], s);
                        const float q = sigmoidf_fast(s);
                        g[K - 1][e] *= q * fmaf(s, 1.f - q, 1.f);
                    }
                    g[K - 1][e] = t < len ? g[K - 1][e] : 0.f;
                    if (t < t1 && t < len) {
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][e] = fmaf(g[K - 1][e], win[k][e], dw[k][e]);
                        dw[K][e] += g[K - 1][e];
                    }
                }
                const int u = t - (K - 1);  // g[j] is dpre[u + j]
                if (u >= t0 || (t0 == 0 && dstate)) {
                    float o[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        o[e] = 0.f;
#pragma unroll
                        for (int k = 0; k < K; ++k) o[e] = fmaf(w[k][e], g[K - 1 - k][e], o[e]);
                    }
                    const int j = u + K - 1 - len;  // which of the returned state's inputs this one is
                    if (dlast && j >= 0 && u < len) {
                        float v[V];
                        conv_load<T, V>(dlast + ((long long)b * (K - 1) + j) * a.D + d, v);
#pragma unroll
                        for (int e = 0; e < V; ++e) o[e] += v[e];
                    }
                    if (u >= 0) conv_store<T, V>(dx + ((long long)b * a.L + u) * a.D + d, o);
                    else conv_store<T, V>(dstate + ((long long)b * (K - 1) + u + K - 1) * a.D + d, o);
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) red[e * 256 + threadIdx.x] = dw[k][e];
        __syncthreads();
        if ((int)threadIdx.x < across && inside) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float s = 0.f;
                for (int r = threadIdx.x; r < 256; r += across) s += red[e * 256 + r];
                parts[((long long)group * (K + 1) + k) * a.D + d + e] = s;
            }
        }
    }
}

// parts [groups][K+1][D] -> dw [D][K], dbias [D]; 16 neighbouring outputs per workgroup, a sixteenth of the partials per group of 16 lanes
__global__ __launch_bounds__(256) void conv_finish_kernel(const float* __restrict__ parts, int groups, int D, int K, float* __restrict__ dw,
                                                          float* __restrict__ dbias) {
    __shared__ float red[256];
    const int i = blockIdx.x * 16 + (threadIdx.x & 15), n = (K + 1) * D;
    float s = 0.f;
    if (i < n) {
#pragma unroll 16
        for (int g = threadIdx.x >> 4; g < groups; g += 16) s += parts[(long long)g * n + i];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x < 16 && i < n) {
        s = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) s += red[threadIdx.x + 16 * r];
        const int k = i / D, d = i % D;
        if (k < K) dw[(long long)d * K + k] = s;
        else if (dbias) dbias[d] = s;
    }
}

// one token of every row; the state moves up by one in place
template <typename T, int K, int V>
__global__ __launch_bounds__(256) void causal_conv_step_kernel(const T* __restrict__ x, long long x_row, T* __restrict__ state, ConvArgs a, T* __restrict__ y) {
    const int vecs = a.D / V;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)a.B * vecs) return;
    const int b = (int)(i / vecs), d = (int)(i % vecs) * V;
    float w[K][V], s[V], in[K][V];
    T* at = state + (long long)b * (K - 1) * a.D + d;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) conv_load<T, V>(at + (long long)k * a.D, in[k]);
    conv_load<T, V>(x + b * x_row + d, in[K - 1]);
    conv_weights<K, V>(a, d, w, s);
#pragma unroll
    for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int k = 0; k < K; ++k) s[e] = fmaf(w[k][e], in[k][e], s[e]);
        if (a.silu) s[e] *= sigmoidf_fast(s[e]);
    }
    conv_store<T, V>(y + (long long)b * a.D + d, s);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) conv_store<T, V>(at + (long long)k * a.D, in[k + 1]);
}

static bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 16-byte vectors need every address that is formed from a channel index to be a multiple of 16 bytes
template <typename T>
static int conv_vector(const ConvArgs& a, const void* p0, const void* p1, const void* p2, const void* p3) {
    constexpr int V = 16 / sizeof(T);
    const bool ok = a.D % V == 0 && a.x_row % V == 0 && a.x_tok % V == 0 && on16(a.x) && on16(a.w) && on16(a.bias) && on16(a.state) && on16(p0) && on16(p1) && on16(p2) && on16(p3);
    return ok ? V : 1;
}
// channel vectors per workgroup row: the widest of 64, 32, 16, 8 that leaves no more idle threads than a narrower one would
static void conv_tiles(ConvArgs& a, int vecs) {
    int best = 3;
    for (int t = 4; t <= 6; ++t)
        if (((vecs + (1 << t) - 1) >> t << t) <= ((vecs + (1 << best) - 1) >> best << best)) best = t;
    a.tile_log2 = best;
    a.tiles = (vecs + (1 << best) - 1) >> best;
}
static void conv_runs(ConvArgs& a, int vecs, int longest) {
    // the longest run that still gives every SIMD eight waves to choose from; a shorter one re-reads more of the run before it
    a.run = longest;
    while (a.run > 4 && (long long)a.B * ((a.L + a.run - 1) / a.run) * vecs < 8ll * 64 * 1024) a.run /= 2;
    a.runs = (a.L + a.run - 1) / a.run;
}
// partial rows of the weight gradient: about 2048 workgroups over all channel tiles, so the partials stay below 2 % of a large input
static int conv_groups(int tiles) { return 2048 / tiles + 1; }

template <typename T, int K, int V>
static int conv_fwd(ConvArgs a, void* y, void* last, hipStream_t st) {
    const int vecs = a.D / V;
    conv_tiles(a, vecs);
    conv_runs(a, vecs, 32);
    const long long rows = 256 >> a.tile_log2, blocks = ((long long)a.B * a.runs + rows - 1) / rows * a.tiles;
    if (blocks * 256 > 0xffffffffll) return RTFS_EINVAL;  // threads of a launch
    hipLaunchKernelGGL((causal_conv_kernel<T, K, V>), dim3((unsigned)blocks), dim3(256), 0, st, a, static_cast<T*>(y), static_cast<T*>(last));
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}
template <typename T, int K, int V>
static int conv_bwd(ConvArgs a, const void* dy, const void* dlast, void* dx, void* dstate, float* parts, float* dw, float* dbias, hipStream_t st) {
    const int vecs = a.D / V;
    conv_tiles(a, vecs);
    conv_runs(a, vecs, 32);
    const long long rows = 256 >> a.tile_log2, all = ((long long)a.B * a.runs + rows - 1) / rows;
    const int groups = (int)(all < conv_groups(a.tiles) ? all : conv_groups(a.tiles));
    hipLaunchKernelGGL((causal_conv_bwd_kernel<T, K, V>), dim3(groups * a.tiles), dim3(256), 0, st, a, static_cast<const T*>(dy), static_cast<const T*>(dlast),
                       static_cast<T*>(dx), static_cast<T*>(dstate), parts);
    RTFS_LAUNCH_CHECK();
    hipLaunchKernelGGL(conv_finish_kernel, dim3(((K + 1) * a.D + 15) / 16), dim3(256), 0, st, parts, groups, a.D, K, dw, dbias);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}
template <typename T, int K, int V>
static int conv_step(ConvArgs a, const void* x, void* state, void* y, hipStream_t st) {
    const long long blocks = ((long long)a.B * (a.D / V) + 255) / 256;
    if (blocks * 256 > 0xffffffffll) return RTFS_EINVAL;  // threads of a launch
    hipLaunchKernelGGL((causal_conv_step_kernel<T, K, V>), dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const T*>(x), a.x_row, static_cast<T*>(state), a,
                       static_cast<T*>(y));
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

// type x width x alignment -> template
template <typename T, typename F>
static int conv_width(int K, int V, F f) {
    constexpr int W = 16 / sizeof(T);
#define RTFS_CONV_K(k) \
    case k: return V == 1 ? f(T(), std::integral_constant<int, k>(), std::integral_constant<int, 1>()) : f(T(), std::integral_constant<int, k>(), std::integral_constant<int, W>());
    switch (K) {
        RTFS_CONV_K(1) RTFS_CONV_K(2) RTFS_CONV_K(3) RTFS_CONV_K(4) RTFS_CONV_K(5) RTFS_CONV_K(6) RTFS_CONV_K(7) RTFS_CONV_K(8)
    }
#undef RTFS_CONV_K
    return RTFS_EINVAL;
}

}  // namespace rtfs

using namespace rtfs;

extern "C" {

int rtfs_causal_conv_fwd(const void* x, long long x_row, long long x_tok, const float* w, const float* bias, const void* state, const int* lengths, void* y,
                         void* last, int B, int L, int D, int K, int silu, int type, void* stream) {
    if (!x || !w || !y || B <= 0 || L <= 0 || L > (1 << 30) || D <= 0 || D > (1 << 24) || K < 1 || K > 8 || type < 0 || type > 1) return RTFS_EINVAL;
    const ConvArgs a{x, x_row, x_tok, w, bias, state, lengths, B, L, D, silu, 0, 0, 0, 0};
    auto go = [&](auto t, auto k, auto v) { return conv_fwd<decltype(t), decltype(k)::value, decltype(v)::value>(a, y, last, (hipStream_t)stream); };
    return type == 0 ? conv_width<float>(K, conv_vector<float>(a, y, last, nullptr, nullptr), go)
                     : conv_width<__bf16>(K, conv_vector<__bf16>(a, y, last, nullptr, nullptr), go);
}

int rtfs_causal_conv_bwd_work_floats(int D, int K, int type) {
    if (D <= 0 || D > (1 << 24) || K < 1 || K > 8 || type < 0 || type > 1) return RTFS_EINVAL;
    ConvArgs one{}, wide{};  // with and without 16-byte vectors
    conv_tiles(one, D);
    conv_tiles(wide, (D + (type == 0 ? 3 : 7)) / (type == 0 ? 4 : 8));
    const int a = conv_groups(one.tiles), b = conv_groups(wide.tiles);
    return (a > b ? a : b) * (K + 1) * D;
}

int rtfs_causal_conv_bwd(const void* x, long long x_row, long long x_tok, const float* w, const float* bias, const void* state, const int* lengths,
                         const void* dy, const void* dlast, void* dx, void* dstate, float* dw, float* dbias, float* work, int B, int L, int D, int K, int silu,
                         int type, void* stream) {
    if (!x || !w || !dy || !dx || !dw || !work || B <= 0 || L <= 0 || L > (1 << 30) || D <= 0 || D > (1 << 24) || K < 1 || K > 8 || type < 0 || type > 1) return RTFS_EINVAL;
    const ConvArgs a{x, x_row, x_tok, w, bias, state, lengths, B, L, D, silu, 0, 0, 0, 0};
    auto go = [&](auto t, auto k, auto v) {
        return conv_bwd<decltype(t), decltype(k)::value, decltype(v)::value>(a, dy, dlast, dx, dstate, work, dw, dbias, (hipStream_t)stream);
    };
    return type == 0 ? conv_width<float>(K, conv_vector<float>(a, dy, dlast, dx, dstate), go) : conv_width<__bf16>(K, conv_vector<__bf16>(a, dy, dlast, dx, dstate), go);
}

int rtfs_causal_conv_step(const void* x, long long x_row, void* state, const float* w, const float* bias, void* y, int B, int D, int K, int silu, int type,
                          void* stream) {
    if (!x || !w || !y || (!state && K > 1) || B <= 0 || D <= 0 || D > (1 << 24) || K < 1 || K > 8 || type < 0 || type > 1) return RTFS_EINVAL;
    const ConvArgs a{x, x_row, 0, w, bias, state, nullptr, B, 1, D, silu, 0, 0, 0, 0};
    auto go = [&](auto t, auto k, auto v) { return conv_step<decltype(t), decltype(k)::value, decltype(v)::value>(a, x, state, y, (hipStream_t)stream); };
    return type == 0 ? conv_width<float>(K, conv_vector<float>(a, y, nullptr, nullptr, nullptr), go)
                     : conv_width<__bf16>(K, conv_vector<__bf16>(a, y, nullptr, nullptr, nullptr), go);
}

}  // extern "C"
