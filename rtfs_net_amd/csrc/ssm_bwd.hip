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
    int how_dy;
};

// One workgroup takes a chunk for a group's heads (or a part of them, where rows, chunks and groups are too few): C B^T is formed once, and the gradients of B
// and C are summed over the heads in registers, in order.  Two shares of work per wave:
//   scores: wave w owns tokens 16 (w % 4) .. as the columns j of the score tiles (with eight waves, every other one of their row tiles) - these accumulators
//           are operands of dx as they lie;
//   states: the first half of the waves forms U = dy H, the other V = x G, each for its 16-wide slices of N; the tiles of H and G come from memory as operands.
// P goes through in blocks of 64.  Steps and decays are made for four heads at a time, one per wave, and the per-token sums of four heads are finished at a
// time likewise: on one wave they were a third of a head's time.  x and dy are asked for one block ahead.
// 8 rows of 2048 tokens, 32 heads of 64, N = 128, bf16: 350 us; 2048 rows of 125 tokens, 4 heads of 32, N = 32, fp32: 330 us.  About 1100 vector instructions per head
// and wave, spread evenly (the products with H and G a tenth, the per-token sums 13 %, the stores of dx 5 %), are what bounds it, with the matrix instructions
// a third of the time (the forms of P > 32 run out of registers besides: 2 to 35 of 256 go through scratch, in bf16 and with N > 64); smaller rings for a third wave
// per SIMD were slower.
// What a and d(step) need is summed in fp32 from products of split operands (ssm.h), and so is what dB and dC take from the states. The scores that dB and dC are
// formed of, the weights of dx and G in its product are two bf16 each, the second what rounding to the first leaves: 2^-17 of a factor is lost, next to the results'
// own 2^-9 (dx's as single bf16: 1.12 times its rounding's error; 18 us less of 662 at 8 x 2048 tokens).
constexpr int kRing = 4;  // heads per ring of decays and sums

template <int HALF, int ALT> struct HeadSums {
    float rowZ[4][kQ], lowZ[ALT][kQ], inZ[kQ], diagZ[kQ];  // rows per column tile; columns below their own row tile, within it, on its diagonal
    float dotU[HALF][kQ], dotV[HALF][kQ], diagV[kQ], crossing[4];
};

template <typename T, int NP, int PP> struct GradShare {
    static constexpr int kWaves = NP == 128 ? 8 : 4, kThreads = 64 * kWaves, kHalf = kWaves / 2, kAlt = kWaves / 4;
    static constexpr int kSlices = NP / 16 / kHalf;  // 16-wide tiles of N per wave, neighbours
    static constexpr int kOwn = 4 / kAlt;            // row tiles of the scores per wave: tt = o kAlt + alt
    static constexpr int PB = PP < 64 ? PP : 64;
    typedef Tile<T, kQ, NP, kSwapped> Wide;
    typedef Tile<T, kQ, PB, kInOrder> Slim;
    typedef Tile<T, NP, PB, kDownOnly> States;
    typedef Tile<T, kQ, kQ, kInOrder> Scores;
    typedef HeadSums<kHalf, kAlt> Sums;
    static constexpr int kParts = sizeof(T) == 2 ? 2 : 1;  // bf16: operands that were fp32 (G, scores), and what rounding leaves of them
    // The weights of dx are formed with the first block of P where their registers are to spare, else anew where they are used (2048 rows of 125 tokens, 4 heads of
    // 32, N = 32, fp32: 556 us, 560 formed late; 4 rows of 1024 tokens, 16 heads of 64, N = 128, fp32: 261 us, 272 formed early and spilled).
    static constexpr bool kEarly = NP == 32;
    static constexpr int kMain = 2 * Slim::kBytes + kParts * States::kBytes, kLast = kParts * Scores::kBytes, kPool = kMain > kLast ? kMain : kLast;
    static constexpr int kBytes = 2 * Wide::kBytes + kPool + kRing * (int)(sizeof(Decays) + sizeof(Factors) + sizeof(Sums));
    static constexpr int kWavesPerSimd = kWaves == 8 || kBytes * 2 <= 160 * 1024 ? 2 : 1;
};

// values of four token tiles, summed over the four lane groups g: lane l gets the total of token l
__device__ __forceinline__ float sum_groups(const float (&v)[4]) {
    const int g = (threadIdx.x & 63) >> 4;
    const bool upper = g & 2, odd = g & 1;
    const float a0 = (upper ? v[2] : v[0]) + __shfl_xor(upper ? v[0] : v[2], 32, 64), a1 = (upper ? v[3] : v[1]) + __shfl_xor(upper ? v[1] : v[3], 32, 64);
    return (odd ? a1 : a0) + __shfl_xor(odd ? a0 : a1, 16, 64);
}

template <typename T, int NP, int PP>
__global__ __launch_bounds__((GradShare<T, NP, PP>::kThreads), (GradShare<T, NP, PP>::kWavesPerSimd)) void scan_grad_kernel(GradArgs q) {
    typedef GradShare<T, NP, PP> S;
    typedef T T4 __attribute__((ext_vector_type(4)));
    constexpr int PB = S::PB, NS = S::kSlices, kOwn = S::kOwn;
    __shared__ __attribute__((aligned(16))) typename S::Wide Bs, Cs;
    __shared__ __attribute__((aligned(16))) char pool[S::kPool];
    __shared__ __attribute__((aligned(16))) Decays decays[kRing];
    __shared__ __attribute__((aligned(16))) Factors factors[kRing];
    __shared__ __attribute__((aligned(16))) typename S::Sums sums[kRing];
    typename S::Slim &Ys = *reinterpret_cast<typename S::Slim*>(pool), &Xs = *reinterpret_cast<typename S::Slim*>(pool + S::Slim::kBytes);
    typename S::States* Gs = reinterpret_cast<typename S::States*>(pool + 2 * S::Slim::kBytes);  // rows: places of n
    const ScanArgs& a = q.a;
    unsigned i0 = xcd_block(blockIdx.x, gridDim.x);
    const int part = (int)(i0 % q.parts);
    i0 /= q.parts;
    const int grp = (int)(i0 % a.G);
    i0 /= a.G;
    const int c = (int)(i0 % a.chunks), b = (int)(i0 / a.chunks);
    const int lane = threadIdx.x & 63, w = wave_index(), lc = lane & 15, g = lane >> 4;
    const int len = row_length(a.lengths, b, a.L), t0 = c * kQ, all = a.L - t0 < kQ ? a.L - t0 : kQ, rows = len - t0 < 0 ? 0 : len - t0 < kQ ? len - t0 : kQ;
    const int each = a.H / a.G, h0 = grp * each + part * q.part_heads, h1 = h0 + q.part_heads < (grp + 1) * each ? h0 + q.part_heads : (grp + 1) * each;
    const int blocks = (a.P + PB - 1) / PB;  // of P that hold anything
    const int jt = w & 3, alt = w >> 2, j = 16 * jt + lc;  // this lane's column of the score tiles
    const bool role_v = w >= S::kHalf;
    const int first = role_v ? w - S::kHalf : w, nt0 = first * NS;  // this wave's tiles of N: nt0 and its NS - 1 neighbours
    const typename S::Slim& Rs = role_v ? Xs : Ys;
    const typename S::Wide &Ks = role_v ? Bs : Cs, &Os = role_v ? Cs : Bs;
    const float *mine = role_v ? q.behind : q.front;
    Load<T, PB, 128> ahead;  // x by waves 0 and 1, dy by waves 2 and 3
    auto ask = [&](int h, int p0) {
        const T* src = w < 2 ? static_cast<const T*>(a.x) + b * a.x_row + t0 * a.x_tok : static_cast<const T*>(q.dy) + ((long long)b * a.L + t0) * a.H * a.P;
        if (w < 4)
            ahead.ask(threadIdx.x & 127, src + (long long)h * a.P + p0, w < 2 ? a.x_tok : (long long)a.H * a.P, rows, a.P - p0, w < 2 ? a.how_x : q.how_dy);
    };
    float raw = 0.f;
    auto ask_step = [&](int h) { raw = w < kRing && h + w < h1 && lane < rows ? a.dt.raw(b, t0 + lane, h + w) : 0.f; };
    {
        const T* Bg = static_cast<const T*>(a.B) + b * a.b_row + t0 * a.b_tok + (long long)grp * a.N;
        const T* Cg = static_cast<const T*>(a.C) + b * a.c_row + t0 * a.c_tok + (long long)grp * a.N;
        Load<T, NP, S::kThreads> lb, lcc;
        lb.ask(threadIdx.x, Bg, a.b_tok, rows, a.N, a.how_b);
        lcc.ask(threadIdx.x, Cg, a.c_tok, rows, a.N, a.how_c);
        ask(h0, 0), ask_step(h0);
        lb.put(threadIdx.x, Bs), lcc.put(threadIdx.x, Cs);
    }
    __syncthreads();
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const typename S::Wide::Lane ln;
    const typename S::Slim::Lane lp;
    const typename S::States::Lane lg;
    f32x4 cb[4], dcb[kOwn], sum[4][NS];  // rows t, columns j; rows n, columns t
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
        cb[tt] = zero;
        if (tt < kOwn) dcb[tt] = zero;
        if (tt >= jt)
#pragma unroll
            for (int k = 0; k < NP / 32; ++k) cb[tt] = mma(Cs.row(ln, 16 * tt, 32 * k), Bs.row(ln, 16 * jt, 32 * k), cb[tt]);
#pragma unroll
        for (int s = 0; s < NS; ++s) sum[tt][s] = zero;
    }
    for (int h = h0; h < h1; ++h) {
        const int ring = (h - h0) % kRing;
        const Decays& e = decays[ring];
        const Factors& f = factors[ring];
        typename S::Sums& hs = sums[ring];
        const float D = a.D ? a.D[h] : 0.f;
        const long long at = (((long long)b * a.L + t0) * a.H + h) * a.P, tiles = (((long long)b * a.chunks + c) * a.H + h) * PP * NP;
        // E of row tile tt >= jt in this lane's column
        auto decay_tile = [&](int tt) {
            const int t = 16 * tt + 4 * g;
            if (tt > jt) return *reinterpret_cast<const f32x4*>(f.near + t) * f.to(tt)[j];
            const f32x4 th = *reinterpret_cast<const f32x4*>(e.hi + t), tl = *reinterpret_cast<const f32x4*>(e.lo + t);
            const float jh = e.hi[j], jl = e.lo[j];
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = 4 * g + i >= lc ? exp2_fast((th[i] - jh) + (tl[i] - jl)) : 0.f;
            return v;
        };
        f32x4 dM[kOwn], R[4][NS];
        Frag<T> wgt[2][S::kParts];
        auto weigh = [&] {
            const float d = e.step[j];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                f32x4 m[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int tt = 2 * k + r;
                    m[r] = zero;
                    if (tt >= jt) m[r] = cb[tt] * decay_tile(tt) * d;
                }
                wgt[k][0] = frag_of<T>(m[0], m[1]);
                if (S::kParts == 2) wgt[k][1] = frag_of<T>(rest_of(m[0]), rest_of(m[1]));
            }
        };
        f32x4 gh = zero;  // four sums: an error of <G, H> is all the chunk's tokens'
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            if (tt < kOwn) dM[tt] = zero;
#pragma unroll
            for (int s = 0; s < NS; ++s) R[tt][s] = zero;
        }
        for (int pb = 0; pb < blocks; ++pb) {
            const int p0 = pb * PB;
            f32x4 tile[NS][PB / 16];
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int pt = 0; pt < PB / 16; ++pt)  // (the walks leave tiles behind P unwritten)
                    tile[s][pt] = p0 + 16 * pt < a.P ? *reinterpret_cast<const f32x4*>(mine + tiles + ((p0 / 16 + pt) * (NP / 16) + nt0 + s) * 256 + lane * 4) : zero;
            __syncthreads();  // the block before has been read
            if (w < 2) ahead.put(threadIdx.x & 127, Xs);
            else if (w < 4) ahead.put(threadIdx.x & 127, Ys);
            if (pb == 0 && ring == 0) {
                if (w < kRing && h + w < h1) put_factors(factors[w], put_decays(decays[w], raw, lane < rows, a.dt.softplus, a.A[h + w]), 1.f);
                ask_step(h + kRing);
            }
            const bool next = pb + 1 == blocks;  // head
            if (!next || h + 1 < h1) ask(next ? h + 1 : h, next ? 0 : p0 + PB);
            __syncthreads();
            if (S::kEarly && pb == 0) weigh();
#pragma unroll
            for (int k = 0; k < PB / 32; ++k) {
                const Frag<T> xj = Xs.row(lp, 16 * jt, 32 * k);
#pragma unroll
                for (int o = 0; o < kOwn; ++o)
                    if (o * S::kAlt + alt >= jt) dM[o] = mma(Ys.row(lp, 16 * (o * S::kAlt + alt), 32 * k), xj, dM[o]);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                if (role_v) {
#pragma unroll
                    for (int pt = 0; pt < PB / 16; ++pt) {
                        const f32x4 other = p0 + 16 * pt < a.P ? *reinterpret_cast<const f32x4*>(q.front + tiles + ((p0 / 16 + pt) * (NP / 16) + nt0 + s) * 256 + lane * 4) : zero;
                        gh += other * tile[s][pt];
                        Gs[0].put4(16 * (nt0 + s) + lc, 16 * pt + 4 * g, tile[s][pt]);
                        if (S::kParts == 2) Gs[1].put4(16 * (nt0 + s) + lc, 16 * pt + 4 * g, rest_of(tile[s][pt]));
                    }
                }
#pragma unroll
                for (int k = 0; k < PB / 32; ++k) {
                    Split<T> op;
                    split(tile[s][2 * k], tile[s][2 * k + 1], op);
#pragma unroll
                    for (int tt = 0; tt < 4; ++tt) R[tt][s] = mma(op, Rs.row(lp, 16 * tt, 32 * k), R[tt][s]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (next) {
                // per-token sums: over j (16 lanes, and the waves) for the rows, over t (this wave's registers) for the columns
                float low = 0.f, in = 0.f, diag = 0.f, dv = 0.f;
                const float dj = e.step[j];
#pragma unroll
                for (int o = 0; o < kOwn; ++o) {
                    const int tt = o * S::kAlt + alt;
                    f32x4 r = zero;
                    if (tt >= jt) {
                        const f32x4 m = dM[o] * decay_tile(tt), z = m * (S::kAlt == 1 ? cb[o] : alt ? cb[(2 * o + 1) & 3] : cb[2 * o & 3]);
                        dcb[o] += m * dj;
                        r = z * dj;
                        if (tt > jt) {
                            low += (z[0] + z[1]) + (z[2] + z[3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const bool on = 4 * g + i == lc;
                                in += on ? 0.f : z[i], diag += on ? z[i] : 0.f, dv += on ? dM[o][i] : 0.f;
                                r[i] = on ? 0.f : r[i];
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) r[i] = row16_sum(r[i]);
                    }
                    if (lc == 0) *reinterpret_cast<f32x4*>(hs.rowZ[jt] + 16 * tt + 4 * g) = r;
                }
                low += __shfl_xor(low, 16, 64), in += __shfl_xor(in, 16, 64), diag += __shfl_xor(diag, 16, 64), dv += __shfl_xor(dv, 16, 64);
                low += __shfl_xor(low, 32, 64), in += __shfl_xor(in, 32, 64), diag += __shfl_xor(diag, 32, 64), dv += __shfl_xor(dv, 32, 64);
                if (g == 0) {
                    hs.lowZ[alt][j] = low;
                    if (jt % S::kAlt == alt) hs.inZ[j] = in, hs.diagZ[j] = diag, hs.diagV[j] = dv;
                }
                float dots[4];
#pragma unroll
                for (int tt = 0; tt < 4; ++tt) {
                    const int t = 16 * tt + lc;
                    const float by = role_v ? e.to[t] * e.step[t] : e.from[t];
                    f32x4 k0, k1, v = zero;
                    widen(Ks.row_any(ln, 16 * tt, 16 * nt0 & ~31), k0, k1);
                    if (NS == 1) k0 = nt0 & 1 ? k1 : k0;
#pragma unroll
                    for (int s = 0; s < NS; ++s) {
                        v += (s == 0 ? k0 : k1) * R[tt][s];
                        sum[tt][s] += R[tt][s] * by;
                    }
                    dots[tt] = (v[0] + v[1]) + (v[2] + v[3]);
                }
                (role_v ? hs.dotV : hs.dotU)[first][lane] = sum_groups(dots);
                if (role_v) {
                    const float v = wave_sum((gh[0] + gh[1]) + (gh[2] + gh[3]));
                    if (lane == 0) hs.crossing[first] = v;
                }
            }
            __syncthreads();
            const float end = e.to[j] * e.step[j];
            if (!S::kEarly) weigh();
            T* dx = static_cast<T*>(q.dx) + at + (long long)j * a.H * a.P + p0;
#pragma unroll
            for (int i = 0; i < PB / 16 / S::kAlt; ++i) {
                const int pt = S::kAlt == 1 ? i : 2 * i;  // of two neighbours this wave's is known when it runs
                f32x4 acc = zero;  // rows p, columns j
#pragma unroll
                for (int k = 0; k < NP / 32; ++k)
#pragma unroll
                    for (int m = S::kParts - 1; m >= 0; --m)
                        acc = mma(alt ? Gs[m].down(lg, 32 * k, pt + S::kAlt - 1) : Gs[m].down(lg, 32 * k, pt), Bs.row(ln, 16 * jt, 32 * k), acc);
                acc = acc * end + Ys.get4(j, 16 * (pt + alt) + 4 * g) * D;  // (as a part of the weights D would be rounded with them)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (2 * k + 1 >= jt)
#pragma unroll
                        for (int m = S::kParts - 1; m >= 0; --m) acc = mma(alt ? Ys.down(lp, 32 * k, pt + S::kAlt - 1) : Ys.down(lp, 32 * k, pt), wgt[k][m], acc);
                const int p = 16 * (pt + alt) + 4 * g;
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
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if ((ring == kRing - 1 || h + 1 == h1) && w <= ring) {  // a wave per head of the ring, one token per lane
            const int hw = h - ring + w;
            const Decays& d = decays[w];
            const typename S::Sums& s = sums[w];
            const float step = d.step[lane], A = a.A[hw];
            float u = 0.f, v = 0.f, cross = 0.f, low = 0.f;
#pragma unroll
            for (int i = 0; i < S::kHalf; ++i) u += s.dotU[i][lane], v += s.dotV[i][lane], cross += s.crossing[i];
#pragma unroll
            for (int i = 0; i < S::kAlt; ++i) low += s.lowZ[i][lane];
            u *= d.from[lane], v *= d.to[lane], cross *= d.from[kQ - 1];
            // What crosses token t: sums over tokens in front of it (v) and from it on (u), and sum_{j < t <= t'} Z[t'][j] d[j].  The latter as the rows from t on less
            // the columns from t on would be a small difference of sums whose roundings add up over the chunk, so that only holds within t's own tile; the
            // tiles further away are added, rows of tiles in front of it or columns in front of t.
            const int tile = lane >> 4;
            const float z0 = s.rowZ[0][lane], z1 = s.rowZ[1][lane], z2 = s.rowZ[2][lane], z3 = s.rowZ[3][lane], in = s.inZ[lane];
            const float own = tile == 0 ? z0 : tile == 1 ? z1 : tile == 2 ? z2 : z3, left = tile == 0 ? 0.f : tile == 1 ? z0 : tile == 2 ? z0 + z1 : z0 + z1 + z2;
            const float past1 = wave_sum(tile > 1 ? z0 : 0.f), past2 = wave_sum(tile > 2 ? z0 + z1 : 0.f);  // rows behind tiles 1 and 2 of columns in front of them
            const double near = row_sum_from((double)left + ((double)own - (double)step * in)), below = (double)step * low;
            const double over64 = (double)cross + running_sum_before((double)step * v) + running_sum_from((double)u) + near + (row_sum_to(below) - below);
            const float over = (float)(over64 + (double)(tile == 1 ? past1 : tile == 2 ? past2 : 0.f)), col = in + low;
            float dstep = lane < rows ? fmaf(A, over, col + s.diagZ[lane] + v) : 0.f;
            if (a.dt.softplus) dstep *= -expm1f(-step);  // softplus'(v) = 1 - e^{-softplus(v)}
            if (lane < all) {
                const long long o = ((long long)b * a.L + t0 + lane) * a.H + hw;
                if (a.dt.type == 0) static_cast<float*>(q.ddt)[o] = dstep;
                else static_cast<__bf16*>(q.ddt)[o] = (__bf16)dstep;
            }
            const float sA = wave_sum(lane < rows ? over * step : 0.f), sD = wave_sum(s.diagV[lane]), sb = wave_sum(dstep);
            if (lane == 0) {
                float* o = q.sums + (((long long)b * a.chunks + c) * a.H + hw) * 3;
                o[0] = sA, o[1] = sD, o[2] = sb;
            }
        }
    }
    // dC += (V o E) d B, dB += (V o E)^T d C, summed over the heads before the product
    const typename S::Scores::Lane lq;
    typename S::Scores* Ms = reinterpret_cast<typename S::Scores*>(pool);
    __syncthreads();
#pragma unroll
    for (int o = 0; o < kOwn; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 16 * (o * S::kAlt + alt) + 4 * g + i;
            Ms[0].put(t, j, dcb[o][i]);
            if (S::kParts == 2) Ms[1].put(t, j, dcb[o][i] - (float)(T)dcb[o][i]);
        }
    __syncthreads();
    T* grad = static_cast<T*>(role_v ? q.dB : q.dC);
    float* wide = role_v ? q.pB : q.pC;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const int n = swapped(nt0 + s, 4 * g);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const Frag<T> o = Os.down_any(32 * k, nt0 + s);
#pragma unroll
            for (int tt = 0; tt < 4; ++tt)
#pragma unroll
                for (int m = S::kParts - 1; m >= 0; --m) sum[tt][s] = mma(o, role_v ? Ms[m].down(lq, 32 * k, tt) : Ms[m].row(lq, 16 * tt, 32 * k), sum[tt][s]);
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
            const int t = 16 * tt + lc;
            if (t >= all || n >= a.N) continue;
            const long long o = (((long long)b * a.L + t0 + t) * a.G + grp) * a.N + n;
            const long long ow = (long long)part * a.rows * a.L * a.G * a.N + o;
            T4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (T)sum[tt][s][i];
            if (a.N % 4 == 0) {
                if (q.parts > 1) *reinterpret_cast<f32x4*>(wide + ow) = sum[tt][s];
                else *reinterpret_cast<T4*>(grad + o) = v;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < a.N) {
                        if (q.parts > 1) wide[ow + i] = sum[tt][s][i];
                        else grad[o + i] = v[i];
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

// Workgroups that share a group's heads: as few as fill the chip - two workgroups of four waves per CU, or one of eight (N > 64).  More form C B^T more often and
// leave partial gradients of B and C to be added (8 rows of 2048 tokens, 32 heads of 64, N = 128, one group: 324 us in one part, 328 + 12 us in two).
static void grad_parts(const ScanArgs& a, int& parts, int& heads) {
    const int each = a.H / a.G;
    const long long blocks = (long long)a.rows * a.chunks * a.G;
    const long long full = a.N > 64 ? 256 : 512, want = blocks >= full ? 1 : (full + blocks - 1) / blocks;
    heads = want >= each ? 1 : (int)((each + want - 1) / want);
    parts = (each + heads - 1) / heads;
}

template <typename T, int NP, int PP>
static int launch_grad(const GradArgs& q, hipStream_t st) {
    const long long blocks = (long long)q.a.rows * q.a.chunks * q.a.G * q.parts;
    if (blocks * GradShare<T, NP, PP>::kThreads > 0xffffffffll) return RTFS_EINVAL;  // threads of a launch
    hipLaunchKernelGGL((scan_grad_kernel<T, NP, PP>), dim3((unsigned)blocks), dim3(GradShare<T, NP, PP>::kThreads), 0, st, q);
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

int rtfs_ssm_scan_bwd_parts(int B, int L, int H, int G, int N) {
    if (!scan_sizes(B, L, H, 1, G, N)) return RTFS_EINVAL;
    ScanArgs a{};
    a.rows = B, a.H = H, a.G = G, a.N = N, a.chunks = (L + kQ - 1) / kQ;
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
        type > 1 || dt_type < 0 || dt_type > 1 || !scan_pitch(x_tok) || !scan_pitch(b_tok) || !scan_pitch(c_tok) || !scan_pitch((long long)H * P))
        return RTFS_EINVAL;
    hipStream_t st = (hipStream_t)stream;
    const Steps steps{dt, dt_row, dt_tok, dt_type, dt_bias, softplus};
    GradArgs q{};
    q.a = scan_args(x, x_row, x_tok, steps, A, Bm, b_row, b_tok, C, c_row, c_tok, D, state, lengths, B, L, H, P, G, N, type, 2);
    const long long d_tok = (long long)H * P;
    // the walk back: dy in the place of x, C in the place of B, the last state's gradient in the place of the state
    const ScanArgs back = scan_args(dy, d_tok * L, d_tok, steps, A, C, c_row, c_tok, C, c_row, c_tok, D, dlast, lengths, B, L, H, P, G, N, type, 2);
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
    q.how_dy = back.how_x;
    auto grad = [&]() -> int { RTFS_SSM_DISPATCH(type, N, 32, 128, P, launch_grad, (q, st)); };
    const int rg = grad();
    if (rg != RTFS_OK) return rg;
    hipLaunchKernelGGL(sum_heads_kernel, dim3(3 * H), dim3(256), 0, st, sums, (long long)B * q.a.chunks, H, dA, dD, dbias);
    RTFS_LAUNCH_CHECK();
    return RTFS_OK;
}

}  // extern "C"
