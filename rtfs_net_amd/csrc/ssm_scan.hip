// Selective state-space scan: forward over prompts, its state walks, and the single-token step.
//   d[t] = softplus(dt[t] + bias) or dt[t] + bias;   S[t] = e^{d[t] A} S[t-1] + d[t] x[t] B[t]^T;   y[t] = S[t] C[t] + D x[t]
// per head of P values with its own scalar decay rate A and a P x N state in fp32; B and C [G][N] are shared by H / G neighbouring heads.
// The chunked matrix form (ssm.h) puts the work on the matrix cores: 2 (64 N + 64 P + 2 N P) operations per token and head instead of a 5 N P vector
// recurrence whose exponentials and dependent adds have no matrix form.
#include "ssm.h"

namespace rtfs {
namespace ssm {

// One workgroup: four waves, each with one head's slice of P, all of one group of heads - they share the tiles of B and C in LDS.
struct Place {
    int b, seg, grp, head, p0;
    bool works;  // waves past the group's last slice only help to load
};
__device__ __forceinline__ Place scan_place(const ScanArgs& a, int w) {
    unsigned i = xcd_block(blockIdx.x, gridDim.x);
    Place p;
    const int quad = (int)(i % a.quads);
    i /= a.quads;
    p.grp = (int)(i % a.G);
    i /= a.G;
    p.seg = (int)(i % a.segs);
    p.b = (int)(i / a.segs);
    const int each = a.H / a.G, unit = quad * 4 + w;
    p.works = unit < each * a.slices;
    p.head = p.grp * each + (p.works ? unit / a.slices : 0);
    p.p0 = p.works ? unit % a.slices * a.width : 0;
    return p;
}

// S <- e^{s[63]} S + sum_j (weight[j] x[j]) B[j]^T, with the weights of a forward or a backward walk.  The weighted x, split, is one operand, tokens of B's
// columns the other, each read once; the state's tiles lie rows n (swapped()), columns p (S[n][p], the forward kernel's) or rows p, columns n (S[p][n], the walks').
template <bool N_FIRST, typename T, int NP, int PW, int R, int C>
__device__ __forceinline__ void advance(f32x4 (&S)[R][C], const Tile<T, kQ, PW, kDownOnly>& X, const Tile<T, kQ, NP, kSwapped>& Bs, const Decays& e, bool backwards) {
    constexpr int NT = NP / 16, PT = PW / 16;
    const int g = (threadIdx.x & 63) >> 4;
    const Lanes<T, NP, kSwapped> ln;
    const Lanes<T, PW, kDownOnly> lp;
    const float whole = e.from[kQ - 1];
    constexpr int kSome = PT < 2 ? PT : 2;  // tiles of P at a time: the split x of all four would take the registers of the loads in flight
#pragma unroll
    for (int p0 = 0; p0 < PT; p0 += kSome)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            Split<T> xs[kSome];
            const int t = 32 * k + 4 * g;
            f32x4 wa = *reinterpret_cast<const f32x4*>((backwards ? e.from : e.to) + t), wb = *reinterpret_cast<const f32x4*>((backwards ? e.from : e.to) + t + 16);
            if (!backwards) wa *= *reinterpret_cast<const f32x4*>(e.step + t), wb *= *reinterpret_cast<const f32x4*>(e.step + t + 16);
#pragma unroll
            for (int pt = 0; pt < kSome; ++pt) {
                f32x4 u, v;
                widen(X.down(lp, 32 * k, p0 + pt), u, v);
                split(u * wa, v * wb, xs[pt]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const Frag<T> bt = Bs.down(ln, 32 * k, nt);
#pragma unroll
                for (int term = Split<T>::kTerms - 1; term >= 0; --term)
#pragma unroll
                    for (int pt = 0; pt < kSome; ++pt) {
                        f32x4& s = N_FIRST ? S[nt][p0 + pt] : S[p0 + pt][nt];
                        if (k == 0 && term == Split<T>::kTerms - 1) s *= whole;
                        s = N_FIRST ? mma(bt, xs[pt].part(term), s) : mma(xs[pt].part(term), bt, s);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
}

// ---- forward ----------------------------------------------------------------------------------------------------------------------------------------------
// A wave walks one segment of its slice and keeps the state in its accumulators from chunk to chunk: an accumulator tile is, as it lies, the operand of the
// product with C, so the state never leaves registers.  So do the scores: C B^T of a pair of token tiles, times decay and step (D joins the diagonal), is the
// operand of the product with x.  LDS holds B and C once for four waves and each wave's x; two barriers per chunk.
// 32768 tokens, 32 heads of 64, N = 128, bf16: 205 us (and 84 + 13 us for the segments' starts); 2048 rows of 125 tokens, 4 heads of 32, N = 32, fp32: 149 us, 40 % of
// it fp32 matrix instructions.  Per wave, vector instructions take as long as the matrix ones, and the LDS holds no third wave per SIMD to run under them.
// Roundings (bf16): y's own alone counts. The scores times decay and step (with D on the diagonal) and the state as it enters the product with C are operands of
// two bf16 each, the second what rounding to the first leaves: they lose 2^-17 of a factor where y is rounded by 2^-9. As single bf16 they cost y 1.04 times its
// rounding's error, and 33 us less of the 205 above. The weighted inputs that build the state are split in three (ssm.h), so the state that is handed on
// has fp32's precision.
// An infinity or a NaN in x would reach the tokens in front of it through scores of zero: it is replaced by zero on its way into LDS, and its value of the head
// becomes a NaN from its token on (odd_from).  Finding none costs 2 %.  (Those of B, C and dt meet no zero: tiles that are masked are not multiplied but chosen.)
// Up to kChain segments a row are chained by the kernel itself, from the own states of the segments in front: that reads each of them half kChain times on average,
// where a launch that chains them reads and writes each and has it read once more (8 rows of four segments, 32 heads of 64 x 128: 16 us).
constexpr int kChain = 8;
constexpr float kNan = __builtin_nanf("");
template <typename T, int NP, int PW> struct ScanShare {
    static constexpr int kBytes = 2 * Tile<T, kQ, NP, kSwapped>::kBytes + 4 * (Tile<T, kQ, PW, kDownOnly>::kBytes + (int)(sizeof(Decays) + sizeof(Factors)) + PW * 4);
    // waves per SIMD: two (256 registers each) where a CU's LDS holds as many workgroups, else one
    static constexpr int kWavesPerSimd = kBytes * 2 <= 160 * 1024 ? 2 : 1;
};

template <typename T, int NP, int PW>
__global__ __launch_bounds__(256, (ScanShare<T, NP, PW>::kWavesPerSimd)) void scan_kernel(ScanArgs a, const float* __restrict__ starts,
                                                                                          const float* __restrict__ segment_decays, T* __restrict__ y,
                                                                                          float* __restrict__ last) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int NT = NP / 16, PT = PW / 16;
    constexpr bool kRest = sizeof(T) == 2;
    __shared__ __attribute__((aligned(16))) Tile<T, kQ, NP, kSwapped> Bs, Cs;
    __shared__ __attribute__((aligned(16))) Tile<T, kQ, PW, kDownOnly> Xs[4];
    __shared__ __attribute__((aligned(16))) Decays decays[4];
    __shared__ __attribute__((aligned(16))) Factors factors[4];
    __shared__ __attribute__((aligned(16))) int odd_from[4][PW];
    const int lane = threadIdx.x & 63, w = wave_index(), lc = lane & 15, g = lane >> 4;
    const Place at = scan_place(a, w);
    const int b = at.b, h = at.head, len = row_length(a.lengths, b, a.L), cols = a.P - at.p0;
    const float A = a.A[h], D = a.D ? a.D[h] : 0.f;
    const T* x = static_cast<const T*>(a.x) + b * a.x_row + (long long)h * a.P + at.p0;
    const T* Bg = static_cast<const T*>(a.B) + b * a.b_row + (long long)at.grp * a.N;
    const T* Cg = static_cast<const T*>(a.C) + b * a.c_row + (long long)at.grp * a.N;
    const long long state_at = ((long long)b * a.H + h) * a.P + at.p0;
    Tile<T, kQ, PW, kDownOnly>& X = Xs[w];
    Decays& e = decays[w];
    Factors& f = factors[w];
    const Lanes<T, NP, kSwapped> ln;
    const Lanes<T, PW, kDownOnly> lp;

    const bool by_four = a.N % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(last)) & 15) == 0;  // state rows lie on 16 bytes
    f32x4 S[NT][PT];  // rows n, columns p
    const int tile = padded(a.P) * NP;
    const bool chain = a.segs <= kChain;
    const float* ends = a.segs > 1 ? starts + ((long long)b * a.H + h) * a.segs * tile + at.p0 * NP + lc * NP + swapped(0, 4 * g) : nullptr;
    const float* start = at.seg > 0 && !chain ? ends + (long long)at.seg * tile : nullptr;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) {
            const int p = 16 * pt + lc, n = swapped(nt, 4 * g);
            S[nt][pt] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (start) {
                S[nt][pt] = *reinterpret_cast<const f32x4*>(start + 16 * pt * NP + swapped(nt, 0));
            } else if (a.state && p < cols) {
                const float* from = a.state + (state_at + p) * a.N + n;
                if (by_four) {
                    if (n < a.N) S[nt][pt] = *reinterpret_cast<const f32x4*>(from);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < a.N) S[nt][pt][i] = from[i];
                }
            }
        }

    if (chain) {
#pragma unroll 2
        for (int i = 0; i < at.seg; ++i) {
            const float decay = segment_decays[((long long)b * a.H + h) * a.segs + i];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int pt = 0; pt < PT; ++pt)
                    S[nt][pt] = S[nt][pt] * decay + *reinterpret_cast<const f32x4*>(ends + (long long)i * tile + 16 * pt * NP + swapped(nt, 0));
        }
    }
    const bool wanted = last && at.seg == a.segs - 1;
    const int c0 = at.seg * a.seg_chunks, c_all = c0 + a.seg_chunks < a.chunks ? c0 + a.seg_chunks : a.chunks;
    const int c_len = (len + kQ - 1) / kQ, c1 = c_all < c_len ? c_all : c_len;
    Load<T, NP, 256, kRest> lb, lcc;
    Load<T, PW, 64, kRest> lx;
    float raw = 0.f;
    auto ask = [&](int c) {
        const long long t0 = (long long)c * kQ;
        const int rows = len - t0 < kQ ? (int)(len - t0) : kQ;
        lb.ask(threadIdx.x, Bg + t0 * a.b_tok, a.b_tok, rows, a.N, a.how_b);
        lcc.ask(threadIdx.x, Cg + t0 * a.c_tok, a.c_tok, rows, a.N, a.how_c);
        lx.ask(lane, x + t0 * a.x_tok, a.x_tok, rows, cols, a.how_x);
        raw = lane < rows ? a.dt.raw(b, t0 + lane, h) : 0.f;
    };
    if (c0 < c1) ask(c0);
    for (int c = c0; c < c1; ++c) {
        const int t0 = c * kQ, rows = len - t0 < kQ ? len - t0 : kQ, all = a.L - t0 < kQ ? a.L - t0 : kQ;
        T* out = y + (((long long)b * a.L + t0) * a.H + h) * a.P + at.p0;
        __syncthreads();  // the chunk before has been read
        lb.put(threadIdx.x, Bs), lcc.put(threadIdx.x, Cs);
        const bool odd = __ballot(lx.odd()) != 0;
        if (odd) {
            int l = lane;
            asm volatile("" : "+v"(l));
            if (l < PW) odd_from[w][l] = kQ;
            lx.clear_odd(l, odd_from[w]);
        }
        lx.put(lane, X);
        const Decay d = put_decays(e, raw, lane < rows, a.dt.softplus, A);
        put_factors(f, d, d.step);
        __syncthreads();
        if (at.works) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // token tiles 2 half and 2 half + 1
                // read and convert again what both halves use: kept from the first half, it would take a hundred registers
                asm volatile("" ::: "memory");
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int pt = 0; pt < PT; ++pt) asm volatile("" : "+v"(S[nt][pt]));
                Frag<T> q[2][NP / 32], m[2][2], rest[2][2];
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int k = 0; k < NP / 32; ++k) q[r][k] = Cs.row(ln, 16 * (2 * half + r), 32 * k);
                // scores: lane l holds token t = its column, four tokens j = its rows
#pragma unroll
                for (int kk = 0; kk <= half; ++kk) {
                    f32x4 s[2][2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int ss = 2 * kk + u;
                        s[0][u] = s[1][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < NP / 32; ++k) {
                            const Frag<T> bj = Bs.row(ln, 16 * ss, 32 * k);
                            if (ss <= 2 * half) s[0][u] = mma(bj, q[0][k], s[0][u]);
                            s[1][u] = mma(bj, q[1][k], s[1][u]);
                        }
                        const int j = 16 * ss + 4 * g;
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int tt = 2 * half + r, t = 16 * tt + lc;
                            if (ss < tt) {
                                s[r][u] *= *reinterpret_cast<const f32x4*>(f.to(tt) + j) * f.near[t];
                            } else if (ss == tt) {
                                const f32x4 jh = *reinterpret_cast<const f32x4*>(e.hi + j), jl = *reinterpret_cast<const f32x4*>(e.lo + j);
                                const f32x4 d = *reinterpret_cast<const f32x4*>(e.step + j);
                                const float th = e.hi[t], tl = e.lo[t];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const float v = s[r][u][i] * exp2_fast((th - jh[i]) + (tl - jl[i])) * d[i];
                                    s[r][u][i] = j + i < t ? v : j + i == t ? v + D : 0.f;
                                }
                            }
                        }
                    }
                    m[0][kk] = frag_of<T>(s[0][0], s[0][1]);
                    m[1][kk] = frag_of<T>(s[1][0], s[1][1]);
                    if (kRest) rest[0][kk] = frag_of<T>(rest_of(s[0][0]), rest_of(s[0][1])), rest[1][kk] = frag_of<T>(rest_of(s[1][0]), rest_of(s[1][1]));
                    __builtin_amdgcn_sched_barrier(0);
                }
                constexpr int kSome = PT < 2 ? PT : 2;
#pragma unroll
                for (int p0 = 0; p0 < PT; p0 += kSome) {
                    f32x4 acc[2][kSome];  // rows p, columns t
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int pt = 0; pt < kSome; ++pt) acc[r][pt] = f32x4{0.f, 0.f, 0.f, 0.f};
                    // the state in front of the chunk
#pragma unroll
                    for (int k = 0; k < NP / 32; ++k)
#pragma unroll
                        for (int pt = 0; pt < kSome; ++pt) {
                            const f32x4 upper = S[2 * k][p0 + pt], lower = S[2 * k + 1][p0 + pt];
                            if (kRest) {
                                const Frag<T> s = frag_of<T>(rest_of(upper), rest_of(lower));
                                acc[0][pt] = mma(s, q[0][k], acc[0][pt]);
                                acc[1][pt] = mma(s, q[1][k], acc[1][pt]);
                            }
                            const Frag<T> s = frag_of<T>(upper, lower);
                            acc[0][pt] = mma(s, q[0][k], acc[0][pt]);
                            acc[1][pt] = mma(s, q[1][k], acc[1][pt]);
                        }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float from = e.from[16 * (2 * half + r) + lc];
#pragma unroll
                        for (int pt = 0; pt < kSome; ++pt) acc[r][pt] *= from;
                    }
#pragma unroll
                    for (int kk = 0; kk <= half; ++kk)
#pragma unroll
                        for (int pt = 0; pt < kSome; ++pt) {
                            const Frag<T> xj = X.down(lp, 32 * kk, p0 + pt);
                            acc[0][pt] = mma(xj, m[0][kk], acc[0][pt]);
                            acc[1][pt] = mma(xj, m[1][kk], acc[1][pt]);
                            if (kRest) acc[0][pt] = mma(xj, rest[0][kk], acc[0][pt]), acc[1][pt] = mma(xj, rest[1][kk], acc[1][pt]);
                        }
                    if (odd) {
                        int l = lane;
                        asm volatile("" : "+v"(l));
#pragma unroll
                        for (int pt = 0; pt < kSome; ++pt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int from = odd_from[w][16 * (p0 + pt) + 4 * (l >> 4) + i] - 32 * half - (l & 15);
                                acc[0][pt][i] = from <= 0 ? kNan : acc[0][pt][i], acc[1][pt][i] = from <= 16 ? kNan : acc[1][pt][i];
                            }
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int t = 16 * (2 * half + r) + lc;
                        T* o = out + (long long)t * a.H * a.P + 4 * g;
#pragma unroll
                        for (int pt = 0; pt < kSome; ++pt) {
                            const int p = 16 * (p0 + pt) + 4 * g;
                            if (t < all && p < cols) {
                                T4 v;
#pragma unroll
                                for (int i = 0; i < 4; ++i) v[i] = (T)(t < rows ? acc[r][pt][i] : 0.f);
                                if (a.P % 4 == 0) {
                                    *reinterpret_cast<T4*>(o + 16 * (p0 + pt)) = v;
                                } else {
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        if (p + i < cols) o[16 * (p0 + pt) + i] = v[i];
                                }
                            }
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (c + 1 < c1) ask(c + 1);  // the registers of the products above are free again; the state's products hide the loads
        if (at.works && (c + 1 < c1 || wanted)) {
            advance<true>(S, X, Bs, e, false);
            if (odd) {
                int l = lc;
                asm volatile("" : "+v"(l));
#pragma unroll
                for (int pt = 0; pt < PT; ++pt) {
                    const float v = odd_from[w][16 * pt + l] < kQ ? kNan : 0.f;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) S[nt][pt] += v;
                }
            }
        }
    }
    if (!at.works) return;
    // chunks behind this row's end: nothing but zeros
    for (int c = c0 > c1 ? c0 : c1; c < c_all; ++c) {
        const int t0 = c * kQ, all = a.L - t0 < kQ ? a.L - t0 : kQ, wide = cols < PW ? cols : PW;
        T* out = y + (((long long)b * a.L + t0) * a.H + h) * a.P + at.p0;
        for (int i = lane; i < all * wide; i += 64) out[(long long)(i / wide) * a.H * a.P + i % wide] = (T)0.f;
    }
    if (wanted) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PT; ++pt) {
                const int p = 16 * pt + lc, n = swapped(nt, 4 * g);
                if (p < cols) {
                    float* to = last + (state_at + p) * a.N + n;
                    if (by_four) {
                        if (n < a.N) *reinterpret_cast<f32x4*>(to) = S[nt][pt];
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (n + i < a.N) to[i] = S[nt][pt][i];
                    }
                }
            }
    }
}

// ---- state walks --------------------------------------------------------------------------------------------------------------------------------------------
// The state alone, in either direction:  forwards  S <- e^{s[63]} S + sum_j e^{s[63]-s[j]} d[j] x[j] B[j]^T,  backwards (the gradient of a chunk's last
// state, from the gradient of the next chunk's)  S <- e^{s[63]} S + sum_t e^{s[t]} dy[t] C[t]^T.  `x` and `B` of the arguments are dy and C then.
// Two uses: a first pass over the segments of a row when rows and heads are too few to fill the chip (`ends`, `decays`: each segment's own state from zero,
// which scan_join_kernel chains), and the states in front of every chunk for the gradients (`tiles`: accumulator tiles as they lie, 1 KB each).
// Two walks in one launch (blockIdx.y): the gradients need both directions at once.
// 8 rows of 2048 tokens, 32 heads of 64, N = 128, bf16: 171 us for both directions, 537 MB of tiles written (113 us at a large copy's rate); 2048 rows of 125 tokens,
// 4 heads of 32, N = 32, fp32: 104 us for about 430 MB.  Loads two chunks ahead changed nothing (53 us for 51 in the first pass, fp32 146 us for 128).
template <typename T, int NP, int PW>
__global__ __launch_bounds__(256, 2) void scan_walk_kernel(ScanArgs a0, WalkOut o0, ScanArgs a1, WalkOut o1) {
    constexpr int NT = NP / 16, PT = PW / 16;
    __shared__ __attribute__((aligned(16))) Tile<T, kQ, NP, kSwapped> Bs;
    __shared__ __attribute__((aligned(16))) Tile<T, kQ, PW, kDownOnly> Xs[4];
    __shared__ __attribute__((aligned(16))) Decays decays[4];
    ScanArgs a = a0;
    WalkOut o = o0;
    if (blockIdx.y) a = a1, o = o1;
    const int lane = threadIdx.x & 63, w = wave_index(), lc = lane & 15, g = lane >> 4;
    const Place at = scan_place(a, w);
    const int b = at.b, h = at.head, len = row_length(a.lengths, b, a.L), cols = a.P - at.p0, PP = padded(a.P);
    const float A = a.A[h];
    const T* x = static_cast<const T*>(a.x) + b * a.x_row + (long long)h * a.P + at.p0;
    const T* Bg = static_cast<const T*>(a.B) + b * a.b_row + (long long)at.grp * a.N;
    const long long head = (long long)b * a.H + h, state_at = head * a.P + at.p0;
    const bool chained = o.starts && at.seg > 0;
    Tile<T, kQ, PW, kDownOnly>& X = Xs[w];
    Decays& e = decays[w];

    f32x4 S[PT][NT];  // rows p, columns n
#pragma unroll
    for (int pt = 0; pt < PT; ++pt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int p = 16 * pt + 4 * g, n = swapped(nt, lc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = 0.f;
                if (chained) v = o.starts[(head * a.segs + at.seg) * PP * NP + (at.p0 + p + i) * NP + n];
                else if (!o.ends && a.state && p + i < cols && n < a.N) v = a.state[(state_at + p + i) * a.N + n];
                S[pt][nt][i] = v;
            }
        }
    // step k of the walk is chunk k, or the k-th from the back
    const int k0 = at.seg * a.seg_chunks, k1 = k0 + a.seg_chunks < a.chunks ? k0 + a.seg_chunks : a.chunks;
    auto chunk = [&](int k) { return o.backwards ? a.chunks - 1 - k : k; };
    Load<T, NP, 256> lb;
    Load<T, PW, 64> lx;
    float raw = 0.f;
    double sum = 0.0;
    auto ask = [&](int k) {
        const long long t0 = (long long)chunk(k) * kQ;
        if (t0 >= len) return;
        const int rows = len - t0 < kQ ? (int)(len - t0) : kQ;
        lb.ask(threadIdx.x, Bg + t0 * a.b_tok, a.b_tok, rows, a.N, a.how_b);
        lx.ask(lane, x + t0 * a.x_tok, a.x_tok, rows, cols, a.how_x);
        raw = lane < rows ? a.dt.raw(b, t0 + lane, h) : 0.f;
    };
    // the last chunk's own step is taken if what is behind the segment is asked for
    const bool final = o.last && at.seg == a.segs - 1;
    const int k2 = o.ends || final ? k1 : k1 - 1;
    if (k0 < k2) ask(k0);
    for (int k = k0; k < k1; ++k) {
        const int c = chunk(k), t0 = c * kQ;
        if (o.tiles && at.works) {
            float* to = o.tiles + (((long long)b * a.chunks + c) * a.H + h) * PP * NP + at.p0 * NP + lane * 4;
#pragma unroll
            for (int pt = 0; pt < PT; ++pt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) *reinterpret_cast<f32x4*>(to + (pt * NT + nt) * 256) = S[pt][nt];
        }
        if (k == k2) break;
        __syncthreads();
        if (t0 < len) {
            lb.put(threadIdx.x, Bs), lx.put(lane, X);
            put_decays(e, raw, t0 + lane < len, a.dt.softplus, A);
        }
        if (k + 1 < k2) ask(k + 1);
        __syncthreads();
        if (t0 >= len || !at.works) continue;
        sum += (double)e.hi[kQ - 1] + (double)e.lo[kQ - 1];
        advance<false>(S, X, Bs, e, o.backwards);
    }
    if (!at.works) return;
    float* out = o.ends ? o.ends + (head * a.segs + at.seg) * PP * NP + at.p0 * NP : nullptr;
#pragma unroll
    for (int pt = 0; pt < PT; ++pt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int p = 16 * pt + 4 * g, n = swapped(nt, lc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (out) out[(p + i) * NP + n] = S[pt][nt][i];
                if (final && p + i < cols && n < a.N) o.last[(state_at + p + i) * a.N + n] = S[pt][nt][i];
            }
        }
    if (o.decays && lane == 0 && at.p0 == 0) o.decays[head * a.segs + at.seg] = exp2_fast((float)sum);
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
#pragma unroll 16
    for (int i = 0; i < segs; ++i) {
        const float own = at[i * tile];
        at[i * tile] = s;
        s = fmaf(decays[bh * segs + i], s, own);
    }
}

// ---- one token --------------------------------------------------------------------------------------------------------------------------------------------
// The state is read and written once, 8 N P bytes per head against 6 N P operations: HBM-bound.  Eight lanes share a row of the state (16-byte loads side by
// side, so a wave's load covers eight 128-byte lines), J loads each.  256 rows of 32 heads, 64 x 128 (537 MB of state in and out, partly held by the last-level
// cache): 92 us.
template <typename T, int J>
__global__ __launch_bounds__(256) void scan_step_kernel(const T* __restrict__ x, long long x_row, Steps dt, const float* __restrict__ Av, const T* __restrict__ B,
                                                        long long b_row, const T* __restrict__ C, long long c_row, const float* __restrict__ Dv,
                                                        float* __restrict__ state, T* __restrict__ y, int H, int P, int G, int N, int blocks_p, int by_four) {
    typedef T T4 __attribute__((ext_vector_type(4)));
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
    const T *Bg = B + b * b_row + (long long)grp * N + n0, *Cg = C + b * c_row + (long long)grp * N + n0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int n = n0 + 32 * j;
        bn[j] = cn[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (by_four) {  // (one value at a time, B and C took a third of the kernel's time: 256 rows of 32 heads, 64 x 128: 135 us, now 92)
            if (n < N) bn[j] = __builtin_convertvector(*reinterpret_cast<const T4*>(Bg + 32 * j), f32x4), cn[j] = __builtin_convertvector(*reinterpret_cast<const T4*>(Cg + 32 * j), f32x4);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < N) bn[j][i] = (float)Bg[32 * j + i], cn[j][i] = (float)Cg[32 * j + i];
        }
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

static unsigned scan_groups(const ScanArgs& a) { return (unsigned)a.rows * a.segs * a.G * a.quads; }

template <typename T, int NP, int PW>
static int launch_scan(const ScanArgs& a, const float* starts, void* y, float* last, hipStream_t st) {
    hipLaunchKernelGGL((scan_kernel<T, NP, PW>), dim3(scan_groups(a)), dim3(256), 0, st, a, starts,
                       starts ? starts + (long long)a.rows * a.H * a.segs * (padded(a.P) * NP) : nullptr, static_cast<T*>(y), last);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}
template <typename T, int NP, int PW>
static int launch_walks(const ScanArgs& a0, const WalkOut& o0, const ScanArgs& a1, const WalkOut& o1, int both, hipStream_t st) {
    hipLaunchKernelGGL((scan_walk_kernel<T, NP, PW>), dim3(scan_groups(a0), both ? 2 : 1), dim3(256), 0, st, a0, o0, a1, o1);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

int scan_walks(const ScanArgs& a0, const WalkOut& o0, const ScanArgs& a1, const WalkOut& o1, int both, int type, hipStream_t st) {
    RTFS_SSM_DISPATCH(type, a0.N, 16, 32, a0.width, launch_walks, (a0, o0, a1, o1, both, st));
}

// A wave takes 64, 32 or 16 columns of P: the widest that leaves a group's heads four waves of work (the scores of a head are formed by each of its waves), and
// whose state of N values each fits a wave's registers next to the loads in flight (64 columns of 128 spilled).
// Both sides, 32 heads of 64, N = 64: 32768 tokens, bf16 201 us in 64 columns, 207 in 32; 8 rows of 2048 tokens, bf16 114 and 109 us.  The rule does not look at types:
// fp32, whose tiles of 64 columns leave a CU one workgroup, takes 540 and 279 us, and 462 and 230 in 32 columns.
// Rows are cut into segments, each walked by workgroups of its own, and into no more than 256: a segment's own state is walked first then (B, x and dt read twice,
// the state's products done twice) and the segments' states are chained (about 0.1 us each).  A prompt is cut until every CU has two workgroups (seven rows of
// eight chunks, 6 heads of 48, fp32: 94 us uncut, 75 us in segments of four chunks, 34 us in segments of one).  The gradients' walks, both directions in one
// launch, are cut until every CU has one: they write a tile per chunk and are bound by that, not by the products (8 rows of 2048 tokens, 32 heads of 64, N = 128:
// 172 us uncut at one workgroup per CU; at two 167 us and 118 us more for the first walk and the chain).
void scan_cut(ScanArgs& a, int directions) {
    const int each = a.H / a.G;
    for (a.width = a.P <= 16 ? 16 : a.P <= 32 || a.N > 64 ? 32 : 64; a.width > 16 && each * ((a.P + a.width - 1) / a.width) < 4; a.width /= 2) {}
    a.slices = (a.P + a.width - 1) / a.width;
    a.quads = (each * a.slices + 3) / 4;
    a.chunks = (a.L + kQ - 1) / kQ;
    const long long groups = (long long)a.rows * a.G * a.quads * directions;
    const long long target = directions == 2 ? 256 : 512;
    const long long want = groups >= target ? 1 : (target + groups - 1) / groups;
    const long long per = (a.chunks + want - 1) / want;
    a.seg_chunks = (int)(want == 1 ? a.chunks : per < (a.chunks + 255) / 256 ? (a.chunks + 255) / 256 : per);
    a.segs = (a.chunks + a.seg_chunks - 1) / a.seg_chunks;
}

// Segment starts for the walks and the forward kernel: ws [rows][H][segs][PP * NP] + [rows][H][segs] per direction.
int scan_starts(const ScanArgs& a0, const ScanArgs& a1, const float* state1, float* ws, int both, int type, hipStream_t st) {
    const long long n = (long long)a0.rows * a0.H * a0.segs, tile = padded(a0.P) * padded(a0.N);
    float *e0 = ws, *d0 = ws + n * tile, *e1 = d0 + n, *d1 = e1 + n * tile;
    const WalkOut o0{nullptr, e0, d0, nullptr, nullptr, 0}, o1{nullptr, e1, d1, nullptr, nullptr, 1};
    const int rc = scan_walks(a0, o0, a1, o1, both, type, st);
    if (rc != RTFS_OK || (!both && a0.segs <= kChain)) return rc;  // (the forward kernel chains them itself)
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
    const auto lie = [](const void* p, long long row) { return row % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0; };
    const int by_four = N % 4 == 0 && lie(B, b_row) && lie(C, c_row);
    hipLaunchKernelGGL((scan_step_kernel<T, J>), dim3((unsigned)blocks), dim3(256), 0, st, static_cast<const T*>(x), x_row, dt, A, static_cast<const T*>(B), b_row,
                       static_cast<const T*>(C), c_row, D, state, static_cast<T*>(y), H, P, G, N, blocks_p, by_four);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

}  // namespace ssm
}  // namespace rtfs

using namespace rtfs;
using namespace rtfs::ssm;

extern "C" {

int rtfs_ssm_scan_segments(int B, int L, int H, int P, int G, int N, int directions) {
    if (!scan_sizes(B, L, H, P, G, N) || directions < 1 || directions > 2) return RTFS_EINVAL;
    ScanArgs a{};
    a.rows = B, a.L = L, a.H = H, a.P = P, a.G = G, a.N = N;
    scan_cut(a, directions);
    return a.segs;
}

int rtfs_ssm_tile(int P, int N) { return P <= 0 || P > 128 || N <= 0 || N > 128 ? RTFS_EINVAL : padded(P) * padded(N); }

int rtfs_ssm_scan_fwd(const void* x, long long x_row, long long x_tok, const void* dt, long long dt_row, long long dt_tok, int dt_type, const float* A,
                      const void* Bm, long long b_row, long long b_tok, const void* C, long long c_row, long long c_tok, const float* D, const float* dt_bias,
                      int softplus, const float* state, const int* lengths, void* y, float* last, float* work, int B, int L, int H, int P, int G, int N, int type,
                      void* stream) {
    if (!x || !dt || !A || !Bm || !C || !y || !scan_sizes(B, L, H, P, G, N) || type < 0 || type > 1 || dt_type < 0 || dt_type > 1 ||
        !scan_pitch(x_tok) || !scan_pitch(b_tok) || !scan_pitch(c_tok))
        return RTFS_EINVAL;
    ScanArgs a = scan_args(x, x_row, x_tok, Steps{dt, dt_row, dt_tok, dt_type, dt_bias, softplus}, A, Bm, b_row, b_tok, C, c_row, c_tok, D, state, lengths, B, L, H,
                           P, G, N, type, 1);
    hipStream_t st = (hipStream_t)stream;
    if (a.segs > 1) {
        if (!work) return RTFS_EINVAL;
        const int rc = scan_starts(a, a, nullptr, work, 0, type, st);
        if (rc != RTFS_OK) return rc;
    }
    RTFS_SSM_DISPATCH(type, N, 16, 32, a.width, launch_scan, (a, work, y, last, st));
}

int rtfs_ssm_step(const void* x, long long x_row, const void* dt, long long dt_row, int dt_type, const float* A, const void* Bm, long long b_row, const void* C,
                  long long c_row, const float* D, const float* dt_bias, int softplus, float* state, void* y, int B, int H, int P, int G, int N, int type,
                  void* stream) {
    if (!x || !dt || !A || !Bm || !C || !state || !y || !scan_sizes(B, 1, H, P, G, N) || type < 0 || type > 1 || dt_type < 0 || dt_type > 1 ||
        (reinterpret_cast<uintptr_t>(state) & 15))
        return RTFS_EINVAL;
    const Steps s{dt, dt_row, 0, dt_type, dt_bias, softplus};
    hipStream_t st = (hipStream_t)stream;
#define RTFS_SSM_STEP(T, J) return launch_step<T, J>(x, x_row, s, A, Bm, b_row, C, c_row, D, state, y, B, H, P, G, N, st)
    if (type == 0) {
        if (N <= 32) RTFS_SSM_STEP(float, 1);
        if (N <= 64) RTFS_SSM_STEP(float, 2);
        RTFS_SSM_STEP(float, 4);
    }
    if (N <= 32) RTFS_SSM_STEP(__bf16, 1);
    if (N <= 64) RTFS_SSM_STEP(__bf16, 2);
    RTFS_SSM_STEP(__bf16, 4);
#undef RTFS_SSM_STEP
}

}  // extern "C"
