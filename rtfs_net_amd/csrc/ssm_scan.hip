// Selective state-space scan: forward over prompts, its state walks, and the single-token step.
//   d[t] = softplus(dt[t] + bias) or dt[t] + bias;   S[t] = e^{d[t] A} S[t-1] + d[t] x[t] B[t]^T;   y[t] = S[t] C[t] + D x[t]
// per head of P values with its own scalar decay rate A and a P x N state in fp32; B and C [G][N] are shared by H / G neighbouring heads.
// The chunked matrix form (ssm.h) puts the work on the matrix cores: 2 (64 N + 64 P + 2 N P) operations per token and head instead of a 5 N P vector
// recurrence whose exponentials and dependent adds have no matrix form.
#include "ssm.h"

namespace rtfs {
namespace ssm {

// Which segment of which row and head: heads are innermost (they share B and C), so an XCD's L2 sees one stretch of them.
__device__ __forceinline__ void scan_place(const ScanArgs& a, int& b, int& seg, int& h) {
    const unsigned i = xcd_block(blockIdx.x, gridDim.x);
    h = (int)(i % a.H);
    seg = (int)(i / a.H % a.segs);
    b = (int)(i / a.H / a.segs);
}

// ---- forward ----------------------------------------------------------------------------------------------------------------------------------------------
// One workgroup walks one segment of one head.  Wave w owns 16 (P = 128: 32) of the P columns for all N and keeps their part of the state in its accumulators
// from chunk to chunk: an accumulator tile is, as it lies, the operand of the product with C (the "pair" order), so the state never leaves registers.
// C B^T is shared out by tiles of the lower triangle and meets the decays on its way to LDS; D joins its diagonal.
// Roundings (bf16): the scores times decay and step, and the state as it enters the product with C, once each to bf16 - y is rounded to that anyway; the
// weighted inputs that build the state are kept as two bf16 (ssm.h), so the state that is handed on is good to 2^-17.
template <typename T, int NP, int PP> struct ScanTiles {
    static constexpr int kN = pitch<T>(NP), kP = pitch<T>(PP), kT = pitch<T>(kQ);
    static constexpr int kBt = kTwice<T> ? NP * kT : 0, kX = kTwice<T> ? PP * kT : kQ * kP;
    static constexpr int kBytes = (2 * kQ * kN + kBt + kX + kQ * kT) * (int)sizeof(T) + Waves<PP>::kWaves * (int)sizeof(Decays);
    // waves per SIMD: two (256 registers each) where a CU's LDS holds as many workgroups, else one
    static constexpr int kWavesPerSimd = kBytes * 2 <= 160 * 1024 ? 2 : 1;
};

template <typename T, int NP, int PP>
__global__ __launch_bounds__(Waves<PP>::kThreads, (ScanTiles<T, NP, PP>::kWavesPerSimd)) void scan_kernel(ScanArgs a, const float* __restrict__ starts,
                                                                                                         T* __restrict__ y, float* __restrict__ last) {
    typedef Waves<PP> W;
    typedef ScanTiles<T, NP, PP> S_;
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int kN = S_::kN, kP = S_::kP, kT = S_::kT;
    __shared__ __attribute__((aligned(16))) T Bs[kQ * kN], Cs[kQ * kN], Bt[S_::kBt + 1], Xs[S_::kX], Ms[kQ * kT];
    __shared__ __attribute__((aligned(16))) Decays decays[W::kWaves];
    int b, seg, h;
    scan_place(a, b, seg, h);
    const int lane = threadIdx.x & 63, w = wave_index(), lc = lane & 15, g = lane >> 4;
    const int len = row_length(a.lengths, b, a.L);
    const float A = a.A[h], D = a.D ? a.D[h] : 0.f;
    const T* x = static_cast<const T*>(a.x) + b * a.x_row + (long long)h * a.P;
    const T* Bg = static_cast<const T*>(a.B) + b * a.b_row + (long long)(h / (a.H / a.G)) * a.N;
    const T* Cg = static_cast<const T*>(a.C) + b * a.c_row + (long long)(h / (a.H / a.G)) * a.N;

    f32x4 S[NP / 16][W::kTiles];  // rows n, columns p
#pragma unroll
    for (int nt = 0; nt < NP / 16; ++nt)
#pragma unroll
        for (int pt = 0; pt < W::kTiles; ++pt) {
            const int p = 16 * (w * W::kTiles + pt) + lc, n = 16 * nt + 4 * g;
            S[nt][pt] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (seg > 0) {
                S[nt][pt] = *reinterpret_cast<const f32x4*>(starts + (((long long)b * a.H + h) * a.segs + seg) * PP * NP + p * NP + n);
            } else if (a.state && p < a.P) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < a.N) S[nt][pt][i] = a.state[(((long long)b * a.H + h) * a.P + p) * a.N + n + i];
            }
        }
    for (int i = threadIdx.x; i < kQ * kT; i += W::kThreads) Ms[i] = (T)0.f;

    const int c0 = seg * a.seg_chunks, c_all = c0 + a.seg_chunks < a.chunks ? c0 + a.seg_chunks : a.chunks;
    const int c_len = (len + kQ - 1) / kQ, c1 = c_all < c_len ? c_all : c_len;
    Tile<T, NP, W::kThreads> tb, tc;
    Tile<T, PP, W::kThreads> tx;
    float raw = 0.f;
    auto ask = [&](int c) {
        const long long t0 = (long long)c * kQ;
        const int rows = len - t0 < kQ ? (int)(len - t0) : kQ;
        tb.load(threadIdx.x, Bg + t0 * a.b_tok, a.b_tok, rows, a.N, a.fast_b);
        tc.load(threadIdx.x, Cg + t0 * a.c_tok, a.c_tok, rows, a.N, a.fast_c);
        tx.load(threadIdx.x, x + t0 * a.x_tok, a.x_tok, rows, a.P, a.fast_x);
    };
    auto ask_step = [&](int c) {  // the steps of as many chunks as there are waves, one chunk per wave
        const int t = (c + w) * kQ + lane;
        raw = t < len ? a.dt.raw(b, t, h) : 0.f;
    };
    if (c0 < c1) ask(c0), ask_step(c0);
    for (int c = c0; c < c1; ++c) {
        const int t0 = c * kQ, rows = len - t0 < kQ ? len - t0 : kQ, all = a.L - t0 < kQ ? a.L - t0 : kQ, which = (c - c0) % W::kWaves;
        T* out = y + (((long long)b * a.L + t0) * a.H + h) * a.P;
        __syncthreads();  // the chunk before has been read
        tb.rows(threadIdx.x, Bs), tc.rows(threadIdx.x, Cs);
        if constexpr (kTwice<T>) tb.columns(threadIdx.x, Bt), tx.columns(threadIdx.x, Xs);
        else tx.rows(threadIdx.x, Xs);
        if (which == 0) {
            put_decays(decays[w], raw, (c + w) * kQ + lane < len, a.dt.softplus, A);
            if (c + W::kWaves < c1) ask_step(c + W::kWaves);
        }
        if (c + 1 < c1) ask(c + 1);
        __syncthreads();
        const Decays& e = decays[which];
        // scores of the tiles on and below the diagonal: lane l holds token t = its column, four tokens j = its rows
        for (int i = w; i < 10; i += W::kWaves) {
            const int tt = i < 1 ? 0 : i < 3 ? 1 : i < 6 ? 2 : 3, ss = i - tt * (tt + 1) / 2;
            f32x4 m = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NP / 32; ++k)
                m = mma(frag(Bs + (16 * ss + lc) * kN + 32 * k + 8 * g), frag(Cs + (16 * tt + lc) * kN + 32 * k + 8 * g), m);
            const int t = 16 * tt + lc, j = 16 * ss + 4 * g;
            const float th = e.hi[t], tl = e.lo[t];
            const f32x4 jh = *reinterpret_cast<const f32x4*>(e.hi + j), jl = *reinterpret_cast<const f32x4*>(e.lo + j), d = *reinterpret_cast<const f32x4*>(e.step + j);
            T4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float s = m[i] * exp2_fast((th - jh[i]) + (tl - jl[i])) * d[i];
                v[i] = (T)(j + i < t ? s : j + i == t ? s + D : 0.f);
            }
            *reinterpret_cast<T4*>(Ms + t * kT + j) = v;
        }
        f32x4 acc[W::kTiles][4];  // rows p, columns t
#pragma unroll
        for (int pt = 0; pt < W::kTiles; ++pt)
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) acc[pt][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NP / 32; ++k) {
            Frag<T> s[W::kTiles];
#pragma unroll
            for (int pt = 0; pt < W::kTiles; ++pt) s[pt] = frag_of<T>(S[2 * k][pt], S[2 * k + 1][pt]);
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                const Frag<T> q = frag(Cs + (16 * tt + lc) * kN + 32 * k + 4 * g, Cs + (16 * tt + lc) * kN + 32 * k + 16 + 4 * g);
#pragma unroll
                for (int pt = 0; pt < W::kTiles; ++pt) acc[pt][tt] = mma(s[pt], q, acc[pt][tt]);
            }
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            const float f = e.from[16 * tt + lc];
#pragma unroll
            for (int pt = 0; pt < W::kTiles; ++pt) acc[pt][tt] *= f;
        }
        // the state, before the barrier that the scores wait for
        const float whole = e.from[kQ - 1];
#pragma unroll
        for (int pt = 0; pt < W::kTiles; ++pt) {
            Split<T> xs[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                f32x4 u, v;
                widen(frag_down(Xs, kP, Xs, 16 * (w * W::kTiles + pt) + lc, 32 * k + 8 * g), u, v);
                const float *to = e.to + 32 * k + 8 * g, *d = e.step + 32 * k + 8 * g;
                u *= *reinterpret_cast<const f32x4*>(to) * *reinterpret_cast<const f32x4*>(d);
                v *= *reinterpret_cast<const f32x4*>(to + 4) * *reinterpret_cast<const f32x4*>(d + 4);
                split(u, v, xs[k]);
            }
#pragma unroll
            for (int nt = 0; nt < NP / 16; ++nt) {
                f32x4 s = S[nt][pt] * whole;
#pragma unroll
                for (int k = 0; k < 2; ++k) s = mma(frag_down(Bs, kN, Bt, 16 * nt + lc, 32 * k + 8 * g), xs[k], s);
                S[nt][pt] = s;
            }
        }
        __syncthreads();
#pragma unroll
        for (int pt = 0; pt < W::kTiles; ++pt) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Frag<T> q = frag_down(Xs, kP, Xs, 16 * (w * W::kTiles + pt) + lc, 32 * k + 8 * g);
#pragma unroll
                for (int tt = 2 * k; tt < 4; ++tt) acc[pt][tt] = mma(q, frag(Ms + (16 * tt + lc) * kT + 32 * k + 8 * g), acc[pt][tt]);
            }
            const int p = 16 * (w * W::kTiles + pt) + 4 * g;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                const int t = 16 * tt + lc;
                if (t < all && p < a.P) {
                    T4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = (T)(t < rows ? acc[pt][tt][i] : 0.f);
                    T* o = out + (long long)t * a.H * a.P + p;
                    if (a.P % 4 == 0) {
                        *reinterpret_cast<T4*>(o) = v;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (p + i < a.P) o[i] = v[i];
                    }
                }
            }
        }
    }
    // chunks behind this row's end: nothing but zeros
    for (int c = c0 > c1 ? c0 : c1; c < c_all; ++c) {
        const int t0 = c * kQ, all = a.L - t0 < kQ ? a.L - t0 : kQ;
        T* out = y + (((long long)b * a.L + t0) * a.H + h) * a.P;
        for (int i = threadIdx.x; i < all * a.P; i += W::kThreads) out[(long long)(i / a.P) * a.H * a.P + i % a.P] = (T)0.f;
    }
    if (last && seg == a.segs - 1) {
#pragma unroll
        for (int nt = 0; nt < NP / 16; ++nt)
#pragma unroll
            for (int pt = 0; pt < W::kTiles; ++pt) {
                const int p = 16 * (w * W::kTiles + pt) + lc, n = 16 * nt + 4 * g;
                if (p < a.P) {
                    float* o = last + (((long long)b * a.H + h) * a.P + p) * a.N + n;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < a.N) o[i] = S[nt][pt][i];
                }
            }
    }
}

// ---- state walks --------------------------------------------------------------------------------------------------------------------------------------------
// The state alone, in either direction:  forwards  S <- e^{s[63]} S + sum_j e^{s[63]-s[j]} d[j] x[j] B[j]^T,  backwards (the gradient of a chunk's last
// state, from the gradient of the next chunk's)  S <- e^{s[63]} S + sum_t e^{s[t]} dy[t] C[t]^T.  `x` and `B` of the arguments are dy and C then.
// Two uses: a first pass over the segments of a row when rows and heads are too few to fill the chip (`ends`, `decays`: each segment's own state from zero,
// which scan_join_kernel chains), and the states in front of every chunk for the gradients (`tiles`: accumulator tiles as they lie, 1 KB each).
template <typename T, int NP, int PP> struct WalkTiles {
    static constexpr int kN = pitch<T>(NP), kP = pitch<T>(PP), kT = pitch<T>(kQ);
    static constexpr int kB = kTwice<T> ? NP * kT : kQ * kN, kX = kTwice<T> ? PP * kT : kQ * kP;
};

// two walks in one launch (blockIdx.y): the gradients need both directions at once
template <typename T, int NP, int PP>
__global__ __launch_bounds__(Waves<PP>::kThreads, 2) void scan_walk_kernel(ScanArgs a0, WalkOut o0, ScanArgs a1, WalkOut o1) {
    typedef Waves<PP> W;
    constexpr int kN = pitch<T>(NP), kP = pitch<T>(PP);
    __shared__ __attribute__((aligned(16))) T Bs[WalkTiles<T, NP, PP>::kB], Xs[WalkTiles<T, NP, PP>::kX];
    __shared__ __attribute__((aligned(16))) Decays decays[W::kWaves];
    ScanArgs a = a0;
    WalkOut o = o0;
    if (blockIdx.y) a = a1, o = o1;
    int b, seg, h;
    scan_place(a, b, seg, h);
    const int lane = threadIdx.x & 63, w = wave_index(), lc = lane & 15, g = lane >> 4;
    const int len = row_length(a.lengths, b, a.L);
    const float A = a.A[h];
    const T* x = static_cast<const T*>(a.x) + b * a.x_row + (long long)h * a.P;
    const T* Bg = static_cast<const T*>(a.B) + b * a.b_row + (long long)(h / (a.H / a.G)) * a.N;
    const bool chained = o.starts && seg > 0;

    f32x4 S[W::kTiles][NP / 16];  // rows p, columns n
#pragma unroll
    for (int pt = 0; pt < W::kTiles; ++pt)
#pragma unroll
        for (int nt = 0; nt < NP / 16; ++nt) {
            const int p = 16 * (w * W::kTiles + pt) + 4 * g, n = 16 * nt + lc;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = 0.f;
                if (chained) v = o.starts[(((long long)b * a.H + h) * a.segs + seg) * PP * NP + (p + i) * NP + n];
                else if (!o.ends && a.state && p + i < a.P && n < a.N) v = a.state[(((long long)b * a.H + h) * a.P + p + i) * a.N + n];
                S[pt][nt][i] = v;
            }
        }
    // step k of the walk is chunk k, or the k-th from the back
    const int k0 = seg * a.seg_chunks, k1 = k0 + a.seg_chunks < a.chunks ? k0 + a.seg_chunks : a.chunks;
    auto chunk = [&](int k) { return o.backwards ? a.chunks - 1 - k : k; };
    Tile<T, NP, W::kThreads> tb;
    Tile<T, PP, W::kThreads> tx;
    float raw = 0.f;
    double sum = 0.0;
    auto ask = [&](int k) {
        const long long t0 = (long long)chunk(k) * kQ;
        if (t0 >= len) return;
        const int rows = len - t0 < kQ ? (int)(len - t0) : kQ;
        tb.load(threadIdx.x, Bg + t0 * a.b_tok, a.b_tok, rows, a.N, a.fast_b);
        tx.load(threadIdx.x, x + t0 * a.x_tok, a.x_tok, rows, a.P, a.fast_x);
    };
    auto ask_step = [&](int k) {
        const long long t = (long long)chunk(k + w) * kQ + lane;
        raw = k + w < k1 && t < len ? a.dt.raw(b, t, h) : 0.f;
    };
    ask(k0), ask_step(k0);
    for (int k = k0; k < k1; ++k) {
        const int c = chunk(k), t0 = c * kQ, which = (k - k0) % W::kWaves;
        if (o.tiles) {
            float* to_tile = o.tiles + (((long long)b * a.chunks + c) * a.H + h) * PP * NP;
#pragma unroll
            for (int pt = 0; pt < W::kTiles; ++pt)
#pragma unroll
                for (int nt = 0; nt < NP / 16; ++nt)
                    *reinterpret_cast<f32x4*>(to_tile + ((w * W::kTiles + pt) * (NP / 16) + nt) * 256 + lane * 4) = S[pt][nt];
        }
        __syncthreads();
        if (t0 < len) {
            if constexpr (kTwice<T>) tb.columns(threadIdx.x, Bs), tx.columns(threadIdx.x, Xs);
            else tb.rows(threadIdx.x, Bs), tx.rows(threadIdx.x, Xs);
        }
        if (which == 0) {
            put_decays(decays[w], raw, k + w < k1 && (long long)chunk(k + w) * kQ + lane < len, a.dt.softplus, A);
            if (k + W::kWaves < k1) ask_step(k + W::kWaves);
        }
        if (k + 1 < k1) ask(k + 1);
        __syncthreads();
        if (t0 >= len) continue;
        const Decays& e = decays[which];
        sum += (double)e.hi[kQ - 1] + (double)e.lo[kQ - 1];
        const float whole = e.from[kQ - 1];
#pragma unroll
        for (int pt = 0; pt < W::kTiles; ++pt) {
            Split<T> xs[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                f32x4 u, v;
                widen(frag_down(Xs, kP, Xs, 16 * (w * W::kTiles + pt) + lc, 32 * q + 8 * g), u, v);
                const int t = 32 * q + 8 * g;
                if (o.backwards) {
                    u *= *reinterpret_cast<const f32x4*>(e.from + t), v *= *reinterpret_cast<const f32x4*>(e.from + t + 4);
                } else {
                    u *= *reinterpret_cast<const f32x4*>(e.to + t) * *reinterpret_cast<const f32x4*>(e.step + t);
                    v *= *reinterpret_cast<const f32x4*>(e.to + t + 4) * *reinterpret_cast<const f32x4*>(e.step + t + 4);
                }
                split(u, v, xs[q]);
            }
#pragma unroll
            for (int nt = 0; nt < NP / 16; ++nt) {
                f32x4 s = S[pt][nt] * whole;
#pragma unroll
                for (int q = 0; q < 2; ++q) s = mma(xs[q], frag_down(Bs, kN, Bs, 16 * nt + lc, 32 * q + 8 * g), s);
                S[pt][nt] = s;
            }
        }
    }
    float* out = o.ends ? o.ends + (((long long)b * a.H + h) * a.segs + seg) * PP * NP : nullptr;
    const bool final = o.last && seg == a.segs - 1;
#pragma unroll
    for (int pt = 0; pt < W::kTiles; ++pt)
#pragma unroll
        for (int nt = 0; nt < NP / 16; ++nt) {
            const int p = 16 * (w * W::kTiles + pt) + 4 * g, n = 16 * nt + lc;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (out) out[(p + i) * NP + n] = S[pt][nt][i];
                if (final && p + i < a.P && n < a.N) o.last[(((long long)b * a.H + h) * a.P + p + i) * a.N + n] = S[pt][nt][i];
            }
        }
    if (o.decays && threadIdx.x == 0) o.decays[((long long)b * a.H + h) * a.segs + seg] = exp2_fast((float)sum);
}

// Chains the segments' own states: ends[i] becomes the state in front of segment i.  One thread per state element walks the segments.
__global__ __launch_bounds__(256) void scan_join_kernel(float* __restrict__ ends0, const float* __restrict__ decays0, const float* __restrict__ state0,
                                                        float* __restrict__ ends1, const float* __restrict__ decays1, const float* __restrict__ state1, int segs,
                                                        int P, int N, int NP) {
    float* ends = blockIdx.z ? ends1 : ends0;
    const float *decays = blockIdx.z ? decays1 : decays0, *state = blockIdx.z ? state1 : state0;
    const long long bh = blockIdx.x, tile = gridDim.y * 256ll;
    const int e = blockIdx.y * 256 + threadIdx.x, p = e / NP, n = e % NP;
    float s = state && p < P && n < N ? state[(bh * P + p) * N + n] : 0.f;
    float* at = ends + bh * segs * tile + e;
#pragma unroll 8
    for (int i = 0; i < segs; ++i) {
        const float own = at[i * tile];
        at[i * tile] = s;
        s = fmaf(decays[bh * segs + i], s, own);
    }
}

// ---- one token --------------------------------------------------------------------------------------------------------------------------------------------
// The state is read and written once, 8 N P bytes per head against 6 N P operations: HBM-bound.  Eight lanes share a row of the state (16-byte loads side by
// side, so a wave's load covers eight 128-byte lines), J loads each; B and C stay in registers over the rows.
template <typename T, int J>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* __restrict__ x, long long x_row, Steps dt, const float* __restrict__ Av, const T* __restrict__ B,
                                                        long long b_row, const T* __restrict__ C, long long c_row, const float* __restrict__ Dv,
                                                        float* __restrict__ state, T* __restrict__ y, int H, int P, int G, int N, int blocks_p) {
    const int pb = blockIdx.x % blocks_p, h = blockIdx.x / blocks_p % H;
    const long long b = blockIdx.x / blocks_p / H;
    const int r = threadIdx.x >> 3, n0 = (threadIdx.x & 7) * 4, grp = h / (H / G), p = pb * 32 + r;
    if (p >= P) return;
    float* at = state + ((b * H + h) * P + p) * N + n0;
    f32x4 s[J], bn[J], cn[J];
    const bool whole = N % 4 == 0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int n = n0 + 32 * j;
        if (whole) {
            s[j] = n < N ? *reinterpret_cast<const f32x4*>(at + 32 * j) : f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = n + i < N ? at[32 * j + i] : 0.f;
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + 32 * j + i;
            bn[j][i] = n < N ? (float)B[b * b_row + (long long)grp * N + n] : 0.f;
            cn[j][i] = n < N ? (float)C[b * c_row + (long long)grp * N + n] : 0.f;
        }
    float d = dt.raw((int)b, 0, h);
    if (dt.softplus) d = softplus(d);
    const float decay = exp2_fast(d * Av[h] * kLog2e), xv = (float)x[b * x_row + (long long)h * P + p], dx = d * xv;
    float acc = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[j][i] = fmaf(decay, s[j][i], dx * bn[j][i]);
            acc = fmaf(s[j][i], cn[j][i], acc);
        }
        const int n = n0 + 32 * j;
        if (whole) {
            if (n < N) *reinterpret_cast<f32x4*>(at + 32 * j) = s[j];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < N) at[32 * j + i] = s[j][i];
        }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
    if ((threadIdx.x & 7) == 0) y[(b * H + h) * P + p] = (T)(acc + (Dv ? Dv[h] * xv : 0.f));
}

template <typename T, int NP, int PP>
static int launch_scan(const ScanArgs& a, const float* starts, void* y, float* last, hipStream_t st) {
    hipLaunchKernelGGL((scan_kernel<T, NP, PP>), dim3((unsigned)a.rows * a.H * a.segs), dim3(Waves<PP>::kThreads), 0, st, a, starts, static_cast<T*>(y), last);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}
template <typename T, int NP, int PP>
static int launch_walks(const ScanArgs& a0, const WalkOut& o0, const ScanArgs& a1, const WalkOut& o1, int both, hipStream_t st) {
    hipLaunchKernelGGL((scan_walk_kernel<T, NP, PP>), dim3((unsigned)a0.rows * a0.H * a0.segs, both ? 2 : 1), dim3(Waves<PP>::kThreads), 0, st, a0, o0, a1, o1);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

int scan_walks(const ScanArgs& a0, const WalkOut& o0, const ScanArgs& a1, const WalkOut& o1, int both, int type, hipStream_t st) {
    RTFS_SSM_DISPATCH(type, a0.N, a0.P, launch_walks, (a0, o0, a1, o1, both, st));
}

// Segments per row.  One workgroup per row and head walks its chunks in order; below two workgroups per CU rows are cut, as far as four chunks per segment, and
// each segment's own state is walked first (B, x and dt read twice, half the products again).
void scan_cut(ScanArgs& a) {
    a.chunks = (a.L + kQ - 1) / kQ;
    const long long work = (long long)a.rows * a.H;
    const long long want = work >= 512 ? 1 : (1024 + work - 1) / work;
    const long long per = (a.chunks + want - 1) / want;
    a.seg_chunks = (int)(want == 1 ? a.chunks : per < 4 ? 4 : per);
    a.segs = (a.chunks + a.seg_chunks - 1) / a.seg_chunks;
}

// Segment starts for the walks and the forward kernel: ws [rows][H][segs][PP * NP] + [rows][H][segs] per direction.
int scan_starts(const ScanArgs& a0, const ScanArgs& a1, const float* state1, float* ws, int both, int type, hipStream_t st) {
    const long long n = (long long)a0.rows * a0.H * a0.segs, tile = padded(a0.P) * padded(a0.N);
    float *e0 = ws, *d0 = ws + n * tile, *e1 = d0 + n, *d1 = e1 + n * tile;
    const WalkOut o0{nullptr, e0, d0, nullptr, nullptr, 0}, o1{nullptr, e1, d1, nullptr, nullptr, 1};
    const int rc = scan_walks(a0, o0, a1, o1, both, type, st);
    if (rc != RTFS_OK) return rc;
    hipLaunchKernelGGL(scan_join_kernel, dim3(a0.rows * a0.H, (unsigned)(tile / 256), both ? 2 : 1), dim3(256), 0, st, e0, d0, a0.state, e1, d1, state1, a0.segs,
                       a0.P, a0.N, padded(a0.N));
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

template <typename T, int J>
static int launch_step(const void* x, long long x_row, const Steps& dt, const float* A, const void* B, long long b_row, const void* C, long long c_row,
                       const float* D, float* state, void* y, int rows, int H, int P, int G, int N, hipStream_t st) {
    const int blocks_p = (P + 31) / 32;
    const long long blocks = (long long)rows * H * blocks_p;
    if (blocks > 0x7fffffffll) return RTFS_EINVAL;
    hipLaunchKernelGGL((scan_step_kernel<T, J>), dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const T*>(x), x_row, dt, A, static_cast<const T*>(B), b_row,
                       static_cast<const T*>(C), c_row, D, state, static_cast<T*>(y), H, P, G, N, blocks_p);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

}  // namespace ssm
}  // namespace rtfs

using namespace rtfs;
using namespace rtfs::ssm;

extern "C" {

int rtfs_ssm_scan_segments(int B, int L, int H) {
    if (B <= 0 || L <= 0 || H <= 0) return RTFS_EINVAL;
    ScanArgs a{};
    a.rows = B, a.L = L, a.H = H;
    scan_cut(a);
    return a.segs;
}

int rtfs_ssm_tile(int P, int N) { return P <= 0 || P > 128 || N <= 0 || N > 128 ? RTFS_EINVAL : padded(P) * padded(N); }

int rtfs_ssm_scan_fwd(const void* x, long long x_row, long long x_tok, const void* dt, long long dt_row, long long dt_tok, int dt_type, const float* A,
                      const void* Bm, long long b_row, long long b_tok, const void* C, long long c_row, long long c_tok, const float* D, const float* dt_bias,
                      int softplus, const float* state, const int* lengths, void* y, float* last, float* work, int B, int L, int H, int P, int G, int N, int type,
                      void* stream) {
    if (!x || !dt || !A || !Bm || !C || !y || !scan_sizes(B, L, H, P, G, N) || type < 0 || type > 1 || dt_type < 0 || dt_type > 1) return RTFS_EINVAL;
    ScanArgs a = scan_args(x, x_row, x_tok, Steps{dt, dt_row, dt_tok, dt_type, dt_bias, softplus}, A, Bm, b_row, b_tok, C, c_row, c_tok, D, state, lengths, B, L, H,
                           P, G, N, type);
    hipStream_t st = (hipStream_t)stream;
    if (a.segs > 1) {
        if (!work) return RTFS_EINVAL;
        const int rc = scan_starts(a, a, nullptr, work, 0, type, st);
        if (rc != RTFS_OK) return rc;
    }
    RTFS_SSM_DISPATCH(type, N, P, launch_scan, (a, work, y, last, st));
}

int rtfs_ssm_step(const void* x, long long x_row, const void* dt, long long dt_row, int dt_type, const float* A, const void* Bm, long long b_row, const void* C,
                  long long c_row, const float* D, const float* dt_bias, int softplus, float* state, void* y, int B, int H, int P, int G, int N, int type,
                  void* stream) {
    if (!x || !dt || !A || !Bm || !C || !state || !y || !scan_sizes(B, 1, H, P, G, N) || type < 0 || type > 1 || dt_type < 0 || dt_type > 1 ||
        (reinterpret_cast<uintptr_t>(state) & 15))
        return RTFS_EINVAL;
    const Steps s{dt, dt_row, 0, dt_type, dt_bias, softplus};
    hipStream_t st = (hipStream_t)stream;
#define RTFS_SSM_STEP(T)                                                                                               do {                                                                                                                   if (N <= 32) return launch_step<T, 1>(x, x_row, s, A, Bm, b_row, C, c_row, D, state, y, B, H, P, G, N, st);         if (N <= 64) return launch_step<T, 2>(x, x_row, s, A, Bm, b_row, C, c_row, D, state, y, B, H, P, G, N, st);         return launch_step<T, 4>(x, x_row, s, A, Bm, b_row, C, c_row, D, state, y, B, H, P, G, N, st);                  } while (0)
    if (type == 0) RTFS_SSM_STEP(float);
    else RTFS_SSM_STEP(__bf16);
#undef RTFS_SSM_STEP
}

}  // extern "C"
