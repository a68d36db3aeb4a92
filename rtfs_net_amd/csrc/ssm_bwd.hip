// Selective state-space scan: gradients.
// With H the state in front of a chunk and G the gradient of the state behind it (both from the walks of ssm_scan.hip), every chunk is independent:
//   E[t][j] = e^{s[t]-s[j]} (j <= t),  V[t][j] = dy[t].x[j],  M = (C B^T) o E
//   dx[j]  = d[j] (sum_t M[t][j] dy[t] + e^{s[63]-s[j]} G B[j]) + D dy[j]
//   dC[t]  = sum_j (V o E)[t][j] d[j] B[j] + e^{s[t]} H^T dy[t],      dB[j] = d[j] (sum_t (V o E)[t][j] C[t] + e^{s[63]-s[j]} G^T x[j])
// and, with u[t] = e^{s[t]} C[t].(H^T dy[t]), v[j] = e^{s[63]-s[j]} B[j].(G^T x[j]), Z = M o V, the gradient of the log decay at token t is what crosses it:
//   a[t] = e^{s[63]} <G, H> + sum_{j < t} d[j] v[j] + sum_{t' >= t} u[t'] + sum_{j < t <= t'} Z[t'][j] d[j]
//   d(step)[t] = A a[t] + v[t] + sum_{t'} Z[t'][t],   dA = sum a[t] d[t],   dD = sum dy[t].x[t].
#include "ssm.h"

namespace rtfs {
namespace ssm {

struct GradArgs {
    ScanArgs a;
    const void* dy;              // [rows][L][H][P]
    const float *front, *behind; // [rows][chunk][head] accumulator tiles of H and G
    void *dx, *ddt, *dB, *dC;
    float *pB, *pC;              // [parts][rows][L][G][N] when the heads of a group are spread over several workgroups
    float* sums;                 // [rows][chunk][head][3]: dA, dD, dbias
    int parts, part_heads;
    int fast_dy;
};

// One workgroup takes a chunk for a group's heads (or a part of them, where rows, chunks and groups are too few): C B^T is formed once, and the gradients of B
// and C are summed over the heads in registers, in order.  Wave w owns tokens 16 w .. 16 w + 15 as the columns j of the score tiles - their accumulators are
// then operands of dx as they lie - and every fourth 16-wide slice of N for the products with H and G, whose tiles it loads from memory as operands.  P goes
// through in blocks of 64.  What a and d(step) need is summed in fp32 from products of split operands (ssm.h); what only dx, dB and dC need is rounded to the
// tensors' type once on its way into a product.
template <typename T, int NP, int PP>
__global__ __launch_bounds__(256) void scan_grad_kernel(GradArgs q) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int PB = PP < 64 ? PP : 64, kN = pitch<T>(NP), kT = pitch<T>(kQ), kP = pitch<T>(PB);
    constexpr int NT = NP / 64 > 0 ? NP / 64 : 1;  // slices of N per wave
    constexpr int kMain = 2 * kQ * kP + PB * kT + PB * kN, kEnd = kQ * kT + NP * kT;
    __shared__ __attribute__((aligned(16))) T Bs[kQ * kN], Cs[kQ * kN], pool[kMain > kEnd ? kMain : kEnd];
    __shared__ __attribute__((aligned(16))) float hi[kQ], lo[kQ], step[kQ], from[kQ], to[kQ];
    __shared__ float rowZ[4][kQ], dotU[4][kQ], dotV[4][kQ], colZ[kQ], diagZ[kQ], diagV[kQ], crossing[4];
    T *Ys = pool, *Xs = Ys + kQ * kP, *Yt = Xs + kQ * kP, *Gt = Yt + PB * kT;
    const ScanArgs& a = q.a;
    unsigned i0 = xcd_block(blockIdx.x, gridDim.x);
    const int part = (int)(i0 % q.parts);
    i0 /= q.parts;
    const int grp = (int)(i0 % a.G);
    i0 /= a.G;
    const int c = (int)(i0 % a.chunks), b = (int)(i0 / a.chunks);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, lc = lane & 15, g = lane >> 4;
    const int len = row_length(a.lengths, b, a.L), t0 = c * kQ, all = a.L - t0 < kQ ? a.L - t0 : kQ, rows = len - t0 < 0 ? 0 : len - t0 < kQ ? len - t0 : kQ;
    const int each = a.H / a.G, h0 = grp * each + part * q.part_heads, h1 = h0 + q.part_heads < (grp + 1) * each ? h0 + q.part_heads : (grp + 1) * each;
    const T* Bg = static_cast<const T*>(a.B) + b * a.b_row + t0 * a.b_tok + (long long)grp * a.N;
    const T* Cg = static_cast<const T*>(a.C) + b * a.c_row + t0 * a.c_tok + (long long)grp * a.N;
    {
        Tile<T, NP, 256> tile;
        tile.load(Bg, a.b_tok, rows, a.N, a.fast_b);
        tile.rows(Bs);
        tile.load(Cg, a.c_tok, rows, a.N, a.fast_c);
        tile.rows(Cs);
    }
    __syncthreads();
    const int j = 16 * w + lc;  // this lane's column of the score tiles
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    f32x4 cb[4], dcb[4], dBa[4][NT], dCa[4][NT];  // rows t, columns j; rows t, columns n
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
        cb[tt] = dcb[tt] = zero;
        if (tt >= w)
#pragma unroll
            for (int k = 0; k < NP / 32; ++k) cb[tt] = mma(frag(Cs + (16 * tt + lc) * kN + 32 * k + 8 * g), frag(Bs + j * kN + 32 * k + 8 * g), cb[tt]);
#pragma unroll
        for (int s = 0; s < NT; ++s) dBa[tt][s] = dCa[tt][s] = zero;
    }
    for (int h = h0; h < h1; ++h) {
        const float A = a.A[h], D = a.D ? a.D[h] : 0.f;
        float raw = 0.f;
        if (w == 0) {
            float d = 0.f, dh, dl;
            if (lane < rows) {
                d = raw = a.dt.raw(b, t0 + lane, h);
                if (a.dt.softplus) d = softplus(d);
            }
            chunk_decay(d, A, dh, dl);
            const float eh = __shfl(dh, 63, 64), el = __shfl(dl, 63, 64);
            hi[lane] = dh, lo[lane] = dl, step[lane] = d, from[lane] = exp2_fast(dh), to[lane] = exp2_fast((eh - dh) + (el - dl));
        }
        const T* x = static_cast<const T*>(a.x) + b * a.x_row + t0 * a.x_tok + (long long)h * a.P;
        const long long at = (((long long)b * a.L + t0) * a.H + h) * a.P, tiles = (((long long)b * a.chunks + c) * a.H + h) * PP * NP;
        f32x4 E[4], dM[4], U[4][NT], V[4][NT];
        Frag<T> wgt[2];
        float gh = 0.f;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            dM[tt] = zero;
#pragma unroll
            for (int s = 0; s < NT; ++s) U[tt][s] = V[tt][s] = zero;
        }
        for (int p0 = 0; p0 < PP; p0 += PB) {
            if (p0 > 0) __syncthreads();
            if (p0 >= a.P) break;
            {
                Tile<T, PB, 256> tile;
                tile.load(static_cast<const T*>(q.dy) + at + p0, (long long)a.H * a.P, rows, a.P - p0, q.fast_dy);
                tile.rows(Ys), tile.columns(Yt);
                tile.load(x + p0, a.x_tok, rows, a.P - p0, a.fast_x);
                tile.rows(Xs);
            }
            f32x4 H[NT][PB / 16], Gr[NT][PB / 16];
#pragma unroll
            for (int s = 0; s < NT; ++s) {
                const int nt = w + 4 * s;
#pragma unroll
                for (int pt = 0; pt < PB / 16; ++pt) {
                    H[s][pt] = Gr[s][pt] = zero;
                    if (NP >= 64 || nt < NP / 16) {
                        const long long o = tiles + ((p0 / 16 + pt) * (NP / 16) + nt) * 256 + lane * 4;
                        H[s][pt] = *reinterpret_cast<const f32x4*>(q.front + o);
                        Gr[s][pt] = *reinterpret_cast<const f32x4*>(q.behind + o);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            gh = fmaf(H[s][pt][i], Gr[s][pt][i], gh);
                            Gt[(16 * pt + 4 * g + i) * kN + 16 * nt + lc] = (T)Gr[s][pt][i];
                        }
                    }
                }
            }
            __syncthreads();
            if (p0 == 0) {
                const float jh = hi[j], jl = lo[j], d = step[j];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int t = 16 * tt + 4 * g + i;
                        E[tt][i] = t >= j ? exp2_fast((hi[t] - jh) + (lo[t] - jl)) : 0.f;
                    }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    f32x4 m[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        m[r] = cb[2 * k + r] * E[2 * k + r] * d;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (16 * (2 * k + r) + 4 * g + i == j) m[r][i] += D;
                    }
                    wgt[k] = frag_of<T>(m[0], m[1]);
                }
            }
#pragma unroll
            for (int k = 0; k < PB / 32; ++k) {
                const Frag<T> xj = frag(Xs + j * kP + 32 * k + 8 * g);
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
                    if (tt >= w) dM[tt] = mma(frag(Ys + (16 * tt + lc) * kP + 32 * k + 8 * g), xj, dM[tt]);
                if (NP >= 64 || w < NP / 16) {
#pragma unroll
                    for (int s = 0; s < NT; ++s) {
                        Split<T> hs, gs;
                        split(H[s][2 * k], H[s][2 * k + 1], hs);
                        split(Gr[s][2 * k], Gr[s][2 * k + 1], gs);
#pragma unroll
                        for (int tt = 0; tt < 4; ++tt) {
                            U[tt][s] = mma(frag(Ys + (16 * tt + lc) * kP + 32 * k + 4 * g, Ys + (16 * tt + lc) * kP + 32 * k + 16 + 4 * g), hs, U[tt][s]);
                            V[tt][s] = mma(frag(Xs + (16 * tt + lc) * kP + 32 * k + 4 * g, Xs + (16 * tt + lc) * kP + 32 * k + 16 + 4 * g), gs, V[tt][s]);
                        }
                    }
                }
            }
            const float end = to[j] * step[j];
            T* dx = static_cast<T*>(q.dx) + at + (long long)j * a.H * a.P + p0;
#pragma unroll
            for (int pt = 0; pt < PB / 16; ++pt) {
                f32x4 acc = zero;  // rows p, columns j
#pragma unroll
                for (int k = 0; k < NP / 32; ++k) acc = mma(frag(Gt + (16 * pt + lc) * kN + 32 * k + 8 * g), frag(Bs + j * kN + 32 * k + 8 * g), acc);
                acc *= end;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (2 * k + 1 >= w) acc = mma(frag(Yt + (16 * pt + lc) * kT + 32 * k + 4 * g, Yt + (16 * pt + lc) * kT + 32 * k + 16 + 4 * g), wgt[k], acc);
                const int p = 16 * pt + 4 * g;
                if (j < all && p0 + p < a.P) {
                    T4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = (T)acc[i];
                    if (a.P % 4 == 0) {
                        *reinterpret_cast<T4*>(dx + p) = v;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (p0 + p + i < a.P) dx[p + i] = v[i];
                    }
                }
            }
        }
        // per-token sums: over j (16 lanes and the waves) for the rows, over t (this wave's registers) for the columns
        float col = 0.f, diag = 0.f, dv = 0.f;
        const float dj = step[j];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            if (tt >= w) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * tt + 4 * g + i;
                    const float e = dM[tt][i] * E[tt][i], z = e * cb[tt][i];
                    dcb[tt][i] = fmaf(e, dj, dcb[tt][i]);
                    if (t == j) diag += z, dv += dM[tt][i];
                    else col += z;
                    const float r = row16_sum(t == j ? 0.f : z * dj);
                    if (lc == 0) rowZ[w][t] = r;
                }
            } else if (lc == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) rowZ[w][16 * tt + 4 * g + i] = 0.f;
            }
        }
        col += __shfl_xor(col, 16, 64), diag += __shfl_xor(diag, 16, 64), dv += __shfl_xor(dv, 16, 64);
        col += __shfl_xor(col, 32, 64), diag += __shfl_xor(diag, 32, 64), dv += __shfl_xor(dv, 32, 64);
        if (g == 0) colZ[j] = col, diagZ[j] = diag, diagV[j] = dv;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 16 * tt + 4 * g + i;
                float u = 0.f, v = 0.f;
                if (NP >= 64 || w < NP / 16) {
#pragma unroll
                    for (int s = 0; s < NT; ++s) {
                        const int n = 16 * (w + 4 * s) + lc;
                        u = fmaf((float)Cs[t * kN + n], U[tt][s][i], u);
                        v = fmaf((float)Bs[t * kN + n], V[tt][s][i], v);
                        dCa[tt][s][i] = fmaf(from[t], U[tt][s][i], dCa[tt][s][i]);
                        dBa[tt][s][i] = fmaf(to[t] * step[t], V[tt][s][i], dBa[tt][s][i]);
                    }
                }
                u = row16_sum(u), v = row16_sum(v);
                if (lc == 0) dotU[w][t] = u, dotV[w][t] = v;
            }
        gh = wave_sum(gh);
        if (lane == 0) crossing[w] = gh;
        __syncthreads();
        if (w == 0) {  // one token per lane
            const float d = step[lane];
            const float r = rowZ[0][lane] + rowZ[1][lane] + rowZ[2][lane] + rowZ[3][lane];
            const float u = from[lane] * (dotU[0][lane] + dotU[1][lane] + dotU[2][lane] + dotU[3][lane]);
            const float v = to[lane] * (dotV[0][lane] + dotV[1][lane] + dotV[2][lane] + dotV[3][lane]);
            const float cross = from[kQ - 1] * (crossing[0] + crossing[1] + crossing[2] + crossing[3]);
            const double in = running_sum((double)(d * v)), out = running_sum((double)u + ((double)r - (double)d * colZ[lane]));
            const double total = __shfl(out, 63, 64);
            const double before = __shfl_up(out, 1, 64), in_before = __shfl_up(in, 1, 64);
            const float over = (float)((double)cross + (lane ? in_before : 0.0) + (total - (lane ? before : 0.0)));
            float dstep = fmaf(A, over, colZ[lane] + diagZ[lane] + v);
            if (lane >= rows) dstep = 0.f;
            if (a.dt.softplus) dstep = dstep / (1.f + expf(-raw));
            if (lane < all) {
                const long long o = ((long long)b * a.L + t0 + lane) * a.H + h;
                if (a.dt.type == 0) static_cast<float*>(q.ddt)[o] = dstep;
                else static_cast<__bf16*>(q.ddt)[o] = (__bf16)dstep;
            }
            const float sA = wave_sum(lane < rows ? over * d : 0.f), sD = wave_sum(diagV[lane]), sb = wave_sum(dstep);
            if (lane == 0) {
                float* s = q.sums + (((long long)b * a.chunks + c) * a.H + h) * 3;
                s[0] = sA, s[1] = sD, s[2] = sb;
            }
        }
        // what the next head writes before its first barrier (steps and decays, by this wave; the P-block tiles) nobody reads any more
    }
    // dC += (V o E) d B, dB += (V o E)^T d C, summed over the heads before the product
    T *Ms = pool, *Kt = pool + kQ * kT;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        __syncthreads();
        Tile<T, NP, 256> tile;
        if (half == 0) tile.load(Bg, a.b_tok, rows, a.N, a.fast_b);
        else tile.load(Cg, a.c_tok, rows, a.N, a.fast_c);
        tile.columns(Kt);
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            T4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = (T)dcb[tt][i];
                if (half == 0) Ms[(16 * tt + 4 * g + i) * kT + j] = v[i];
            }
            if (half == 1) *reinterpret_cast<T4*>(Ms + j * kT + 16 * tt + 4 * g) = v;
        }
        __syncthreads();
        T* grad = static_cast<T*>(half == 0 ? q.dC : q.dB);
        float* wide = half == 0 ? q.pC : q.pB;
#pragma unroll
        for (int s = 0; s < NT; ++s) {
            const int nt = w + 4 * s, n = 16 * nt + lc;
            if (NP < 64 && nt >= NP / 16) break;
#pragma unroll
            for (int tt = 0; tt < 4; ++tt) {
                f32x4 acc = half == 0 ? dCa[tt][s] : dBa[tt][s];
#pragma unroll
                for (int k = 0; k < 2; ++k) acc = mma(frag(Ms + (16 * tt + lc) * kT + 32 * k + 8 * g), frag(Kt + n * kT + 32 * k + 8 * g), acc);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * tt + 4 * g + i;
                    if (t < all && n < a.N) {
                        const long long o = (((long long)b * a.L + t0 + t) * a.G + grp) * a.N + n;
                        if (q.parts > 1) wide[(long long)part * a.rows * a.L * a.G * a.N + o] = acc[i];
                        else grad[o] = (T)acc[i];
                    }
                }
            }
        }
    }
}

// [parts][n] fp32 -> n values, parts in order
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* __restrict__ p0, T* __restrict__ o0, const float* __restrict__ p1, T* __restrict__ o1, int parts,
                                                        long long n) {
    const float* p = blockIdx.y ? p1 : p0;
    T* o = blockIdx.y ? o1 : o0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += 256ll * gridDim.x) {
        float s = 0.f;
        for (int k = 0; k < parts; ++k) s += p[k * n + i];
        o[i] = (T)s;
    }
}

// sums [rows * chunks][H][3] -> dA, dD, dbias [H]; one workgroup per value, fp64, fixed order
__global__ __launch_bounds__(256) void sum_heads_kernel(const float* __restrict__ sums, long long count, int H, float* __restrict__ dA, float* __restrict__ dD,
                                                        float* __restrict__ dbias) {
    __shared__ double red[4];
    const int h = blockIdx.x / 3, k = blockIdx.x % 3;
    float* out = k == 0 ? dA : k == 1 ? dD : dbias;
    if (!out) return;
    double s = 0.0;
#pragma unroll 4
    for (long long i = threadIdx.x; i < count; i += 256) s += (double)sums[(i * H + h) * 3 + k];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) out[h] = (float)(red[0] + red[1] + red[2] + red[3]);
}

// Workgroups that share a group's heads: as few as give the chip two workgroups per CU
static void grad_parts(const ScanArgs& a, int& parts, int& heads) {
    const int each = a.H / a.G;
    const long long blocks = (long long)a.rows * a.chunks * a.G;
    const long long want = blocks >= 512 ? 1 : (512 + blocks - 1) / blocks;
    heads = want >= each ? 1 : (int)((each + want - 1) / want);
    parts = (each + heads - 1) / heads;
}

template <typename T, int NP, int PP>
static int launch_grad(const GradArgs& q, hipStream_t st) {
    const long long blocks = (long long)q.a.rows * q.a.chunks * q.a.G * q.parts;
    if (blocks > 0x7fffffffll) return RTFS_EINVAL;
    hipLaunchKernelGGL((scan_grad_kernel<T, NP, PP>), dim3((unsigned)blocks), dim3(256), 0, st, q);
    RTFS_LAUNCH_CHECK();
    if (q.parts > 1) {
        const long long n = (long long)q.a.rows * q.a.L * q.a.G * q.a.N, wg = (n + 255) / 256;
        hipLaunchKernelGGL((sum_parts_kernel<T>), dim3((unsigned)(wg < 1024 ? wg : 1024), 2), dim3(256), 0, st, q.pB, static_cast<T*>(q.dB), q.pC,
                           static_cast<T*>(q.dC), q.parts, n);
        RTFS_LAUNCH_CHECK();
    }
    return RTFS_OK;
}

}  // namespace ssm
}  // namespace rtfs

using namespace rtfs;
using namespace rtfs::ssm;

extern "C" {

int rtfs_ssm_scan_bwd_parts(int B, int L, int H, int G) {
    if (B <= 0 || L <= 0 || G <= 0 || H <= 0 || H % G) return RTFS_EINVAL;
    ScanArgs a{};
    a.rows = B, a.L = L, a.H = H, a.G = G;
    scan_cut(a);
    int parts, heads;
    grad_parts(a, parts, heads);
    return parts;
}

int rtfs_ssm_scan_bwd(const void* x, long long x_row, long long x_tok, const void* dt, long long dt_row, long long dt_tok, int dt_type, const float* A,
                      const void* Bm, long long b_row, long long b_tok, const void* C, long long c_row, long long c_tok, const float* D, const float* dt_bias,
                      int softplus, const float* state, const int* lengths, const void* dy, const float* dlast, void* dx, void* ddt, float* dA, void* dB, void* dC,
                      float* dD, float* dbias, float* dstate, float* starts, float* front, float* behind, float* parts, float* sums, int B, int L, int H, int P, int G,
                      int N, int type, void* stream) {
    if (!x || !dt || !A || !Bm || !C || !dy || !dx || !ddt || !dA || !dB || !dC || !front || !behind || !sums || !scan_sizes(B, L, H, P, G, N) || type < 0 ||
        type > 1 || dt_type < 0 || dt_type > 1)
        return RTFS_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    const Steps steps{dt, dt_row, dt_tok, dt_type, dt_bias, softplus};
    GradArgs q{};
    q.a = scan_args(x, x_row, x_tok, steps, A, Bm, b_row, b_tok, C, c_row, c_tok, D, state, lengths, B, L, H, P, G, N, type);
    const long long d_tok = (long long)H * P;
    // the walk back: dy in the place of x, C in the place of B, the last state's gradient in the place of the state
    const ScanArgs back = scan_args(dy, d_tok * L, d_tok, steps, A, C, c_row, c_tok, C, c_row, c_tok, D, dlast, lengths, B, L, H, P, G, N, type);
    grad_parts(q.a, q.parts, q.part_heads);
    if ((q.a.segs > 1 && !starts) || (q.parts > 1 && !parts)) return RTFS_EINVAL;
    const long long n = (long long)B * H * q.a.segs, tile = (long long)padded(P) * padded(N);
    if (q.a.segs > 1) {
        const int rc = scan_starts(q.a, back, dlast, starts, 1, type, st);
        if (rc != RTFS_OK) return rc;
    }
    const bool cut = q.a.segs > 1;
    const WalkOut o0{cut ? starts : nullptr, nullptr, nullptr, front, nullptr, 0};
    const WalkOut o1{cut ? starts + n * (tile + 1) : nullptr, nullptr, nullptr, behind, dstate, 1};
    const int rc = scan_walks(q.a, o0, back, o1, 1, type, st);
    if (rc != RTFS_OK) return rc;
    q.dy = dy, q.front = front, q.behind = behind, q.dx = dx, q.ddt = ddt, q.dB = dB, q.dC = dC, q.sums = sums;
    q.pB = parts, q.pC = parts ? parts + (long long)q.parts * B * L * G * N : nullptr;
    q.fast_dy = back.fast_x;
    auto grad = [&]() -> int { RTFS_SSM_DISPATCH(type, N, P, launch_grad, (q, st)); };
    const int rg = grad();
    if (rg != RTFS_OK) return rg;
    hipLaunchKernelGGL(sum_heads_kernel, dim3(3 * H), dim3(256), 0, st, sums, (long long)B * q.a.chunks, H, dA, dD, dbias);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

}  // extern "C"
