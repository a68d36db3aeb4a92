// Device helpers of the selective scan (ssm_scan.hip, ssm_bwd.hip): chunk staging, matrix-core fragments, decays.
//
// A chunk is 64 tokens.  With s[t] = sum_{j <= t} dt[j] A (this head's log decay inside the chunk) everything inside it is a matrix product:
//   y[t]  = sum_{j <= t} (C[t].B[j]) e^{s[t]-s[j]} dt[j] x[j] + e^{s[t]} S_in C[t],     S_out = e^{s[63]} S_in + sum_j e^{s[63]-s[j]} dt[j] x[j] B[j]^T,
// and only S, the P x N state, goes from chunk to chunk.
#pragma once
#include "common.h"

namespace rtfs {
namespace ssm {

constexpr int kQ = 64;  // tokens per chunk

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---- fragments ------------------------------------------------------------------------------------------------------------------------------------------
// One fragment is a 16 x 32 operand of D[16x16] += A[16x32] B[32x16]: lane l holds 8 values of row (A) or column (B) l & 15; which 8 of the 32 products it
// holds is free as long as A and B agree.  Two choices are used, with g = l >> 4: "run" k = 8 g + j, and "pair" k = 4 g + j, 16 + 4 g + j (j < 4), which is
// how two accumulator tiles lie in registers (lane l: column l & 15, rows 4 g + i), so an accumulator becomes an operand without leaving its lane.
// fp32 goes through v_mfma_f32_16x16x4_f32 (exact products, one value per lane and step), bf16 through one v_mfma_f32_16x16x32_bf16.
template <typename T> struct Frag;
template <> struct Frag<float> { f32x4 a, b; };
template <> struct Frag<__bf16> { bf16x8 v; };

__device__ __forceinline__ f32x4 mma(const Frag<float>& x, const Frag<float>& y, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.a[j], y.a[j], c, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.b[j], y.b[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 mma(const Frag<__bf16>& x, const Frag<__bf16>& y, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.v, y.v, c, 0, 0, 0);
}
// 4 + 4 values in the operand type; two runs of four in LDS (8- or 16-byte aligned), or fp32 values rounded to it
__device__ __forceinline__ Frag<float> frag(const float* p, const float* q) {
    return {*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(q)};
}
__device__ __forceinline__ Frag<__bf16> frag(const __bf16* p, const __bf16* q) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p), b = *reinterpret_cast<const bf16x4*>(q);
    return {__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)};
}
// 8 neighbours ("run")
__device__ __forceinline__ Frag<float> frag(const float* p) { return frag(p, p + 4); }
__device__ __forceinline__ Frag<__bf16> frag(const __bf16* p) { return {*reinterpret_cast<const bf16x8*>(p)}; }

template <typename T> __device__ __forceinline__ Frag<T> frag_of(f32x4 a, f32x4 b);
template <> __device__ __forceinline__ Frag<float> frag_of<float>(f32x4 a, f32x4 b) { return {a, b}; }
template <> __device__ __forceinline__ Frag<__bf16> frag_of<__bf16>(f32x4 a, f32x4 b) {
    Frag<__bf16> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = (__bf16)a[j], f.v[4 + j] = (__bf16)b[j];
    return f;
}
// An fp32 operand as the sum of three bf16 (8 bits of mantissa each, error 2^-25 of it): states, what builds them, and the sums that the gradients of dt and A
// are differences of keep fp32's precision for bf16 tensors too.  fp32 operands are themselves.
template <typename T> struct Split { Frag<T> hi, mid, lo; };
template <> struct Split<float> { Frag<float> hi; };
__device__ __forceinline__ void split(f32x4 a, f32x4 b, Split<float>& s) { s.hi = {a, b}; }
__device__ __forceinline__ void split(f32x4 a, f32x4 b, Split<__bf16>& s) {
    s.hi = frag_of<__bf16>(a, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] -= (float)s.hi.v[j], b[j] -= (float)s.hi.v[4 + j];
    s.mid = frag_of<__bf16>(a, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] -= (float)s.mid.v[j], b[j] -= (float)s.mid.v[4 + j];
    s.lo = frag_of<__bf16>(a, b);
}
__device__ __forceinline__ f32x4 mma(const Split<float>& x, const Frag<float>& y, f32x4 c) { return mma(x.hi, y, c); }
__device__ __forceinline__ f32x4 mma(const Split<__bf16>& x, const Frag<__bf16>& y, f32x4 c) { return mma(x.hi, y, mma(x.mid, y, mma(x.lo, y, c))); }
__device__ __forceinline__ f32x4 mma(const Frag<float>& x, const Split<float>& y, f32x4 c) { return mma(x, y.hi, c); }
__device__ __forceinline__ f32x4 mma(const Frag<__bf16>& x, const Split<__bf16>& y, f32x4 c) { return mma(x, y.hi, mma(x, y.mid, mma(x, y.lo, c))); }

__device__ __forceinline__ void widen(const Frag<float>& f, f32x4& a, f32x4& b) { a = f.a, b = f.b; }
__device__ __forceinline__ void widen(const Frag<__bf16>& f, f32x4& a, f32x4& b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (float)f.v[j], b[j] = (float)f.v[4 + j];
}

// ---- staging --------------------------------------------------------------------------------------------------------------------------------------------
// Row pitch of a tile in LDS with `n` values per row: 16 bytes of padding keep the 16-byte alignment and move neighbouring rows to other banks.
template <typename T> __host__ __device__ constexpr int pitch(int n) { return n + 16 / (int)sizeof(T); }

template <typename T> struct Vec8;
template <> struct Vec8<float> {
    f32x4 a, b;
    __device__ __forceinline__ float get(int i) const { return i < 4 ? a[i] : b[i - 4]; }
    __device__ __forceinline__ void set(int i, float v) { if (i < 4) a[i] = v; else b[i - 4] = v; }
};
template <> struct Vec8<__bf16> {
    bf16x8 v;
    __device__ __forceinline__ __bf16 get(int i) const { return v[i]; }
    __device__ __forceinline__ void set(int i, __bf16 x) { v[i] = x; }
};
template <typename T> __device__ __forceinline__ Vec8<T> zero8() {
    Vec8<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.set(i, (T)0.f);
    return v;
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// 8 values at byte offset `at`; an offset past every tensor (bounds are below 2^31) where there are none
__device__ __forceinline__ void buffer_vec8(Vec8<__bf16>& v, __amdgpu_buffer_rsrc_t r, unsigned at, bool any, bool) {
    v.v = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, any ? at : 0x80000000u, 0, 0));
}
__device__ __forceinline__ void buffer_vec8(Vec8<float>& v, __amdgpu_buffer_rsrc_t r, unsigned at, bool any, bool more) {
    v.a = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, any ? at : 0x80000000u, 0, 0));
    v.b = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, more ? at + 16 : 0x80000000u, 0, 0));
}

// A 64-token tile of up to COLS values per token, read by THREADS threads in units of 4 tokens x 8 values; what lies past `rows` tokens or `cols` values is
// zero (never read: a padded batch may hold anything there).  `fast` (addresses and pitches on 16 bytes, `cols` a multiple of 16 bytes): buffer loads, whose
// bounds check supplies the zeros without a branch; else 16-byte loads at any address, and element by element where a unit crosses `cols`.
// The loads stay in flight in `r` until rows() or columns() stores them to LDS: a tile is asked for one chunk ahead.
template <typename T, int COLS, int THREADS>
struct Tile {
    static constexpr int kUnits = 16 * (COLS / 8), kPer = (kUnits + THREADS - 1) / THREADS;
    Vec8<T> r[kPer][4];

    __device__ __forceinline__ void load(int thread, const T* src, long long row, int rows, int cols, bool fast) {
        // formed anew at every call: hoisted out of the chunk loop, the addresses of the element-wise path alone take a hundred registers
        asm volatile("" : "+v"(thread));
        if (fast) {
            // without a token the bound is 0: nothing is read (below 0 it would be no bound at all)
            const int bytes = rows > 0 ? (int)(((rows - 1) * row + cols) * (long long)sizeof(T)) : 0;
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(src), 0, bytes, 0x00027000);
            const unsigned pitch = (unsigned)row * sizeof(T);
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int u = thread + k * THREADS, c = (u >> 4) * 8;
                unsigned at = (u & 15) * 4 * pitch + c * sizeof(T);
#pragma unroll
                for (int i = 0; i < 4; ++i, at += pitch) buffer_vec8(r[k][i], rsrc, at, c < cols, c + 4 < cols);
            }
            return;
        }
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int u = thread + k * THREADS, c = (u >> 4) * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = (u & 15) * 4 + i;
                r[k][i] = zero8<T>();
                if ((kUnits % THREADS == 0 || u < kUnits) && t < rows && c < cols) {
                    const T* p = src + t * row + c;
                    if (c + 8 <= cols) {
                        __builtin_memcpy(&r[k][i], p, sizeof(Vec8<T>));
                    } else {
#pragma unroll
                        for (int j = 0; j < 7; ++j)
                            if (c + j < cols) r[k][i].set(j, p[j]);
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void rows(int thread, T* dst) const {  // dst[token][value]
        constexpr int ld = pitch<T>(COLS);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int u = thread + k * THREADS, c = (u >> 4) * 8, t = (u & 15) * 4;
            if (kUnits % THREADS == 0 || u < kUnits) {
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<Vec8<T>*>(dst + (t + i) * ld + c) = r[k][i];
            }
        }
    }
    __device__ __forceinline__ void columns(int thread, T* dst) const {  // dst[value][token]
        constexpr int ld = pitch<T>(kQ);
        typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const int u = thread + k * THREADS, c = (u >> 4) * 8, t = (u & 15) * 4;
            if (kUnits % THREADS == 0 || u < kUnits) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    T4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] = r[k][i].get(j);
                    *reinterpret_cast<T4*>(dst + (c + j) * ld + t) = v;
                }
            }
        }
    }
};

// A product over tokens needs its operands with 8 neighbouring TOKENS per lane.  bf16 tiles are stored a second time with tokens innermost (16-byte reads);
// fp32 ones are read across their rows, one value at a time: as many bytes per cycle, and LDS for one copy.
template <typename T> constexpr bool kTwice = sizeof(T) == 2;
__device__ __forceinline__ Frag<float> frag_down(const float* rows, int ld, const float*, int col, int t) {
    Frag<float> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.a[j] = rows[(t + j) * ld + col], f.b[j] = rows[(t + 4 + j) * ld + col];
    return f;
}
// the same across the rows of a tile whatever its type (one value at a time: for products outside the loops)
template <typename T>
__device__ __forceinline__ Frag<T> frag_across(const T* rows, int ld, int col, int t) {
    f32x4 a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (float)rows[(t + j) * ld + col], b[j] = (float)rows[(t + 4 + j) * ld + col];
    return frag_of<T>(a, b);
}
// "pair" order: tokens t .. t + 3 and t + 16 .. t + 19
__device__ __forceinline__ Frag<float> frag_down_pair(const float* rows, int ld, const float*, int col, int t) {
    Frag<float> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.a[j] = rows[(t + j) * ld + col], f.b[j] = rows[(t + 16 + j) * ld + col];
    return f;
}
__device__ __forceinline__ Frag<__bf16> frag_down_pair(const __bf16*, int, const __bf16* cols, int col, int t) {
    return frag(cols + col * pitch<__bf16>(kQ) + t, cols + col * pitch<__bf16>(kQ) + t + 16);
}
__device__ __forceinline__ Frag<__bf16> frag_down(const __bf16*, int, const __bf16* cols, int col, int t) { return frag(cols + col * pitch<__bf16>(kQ) + t); }

// this wave's index, known to the compiler to be the same in all its lanes
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---- decays ---------------------------------------------------------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;

// log(1 + e^v), and its derivative
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

struct Steps {
    const void* dt;
    long long row, tok;
    int type;           // 0 fp32, 1 bf16
    const float* bias;  // [H] or none
    int softplus;
    __device__ __forceinline__ float raw(int b, long long t, int h) const {
        const long long i = b * row + t * tok + h;
        const float v = type == 0 ? static_cast<const float*>(dt)[i] : (float)static_cast<const __bf16*>(dt)[i];
        return bias ? v + bias[h] : v;
    }
};

// sums over the tokens up to and including this lane's, in fp64: the differences s[t] - s[j] are what counts, and behind a strong decay both are large
__device__ __forceinline__ double running_sum(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    return v;
}
// One wave, one token per lane: log2 decay (as two floats whose sum is the fp64 value to 48 bits).
__device__ __forceinline__ void chunk_decay(float step, float A, float& hi, float& lo) {
    const double s = running_sum((double)step * (double)A * 1.4426950408889634074);
    hi = (float)s;
    lo = (float)(s - (double)hi);
}
// What the products of a chunk take from its decays, per token: s as two floats, d, e^{s[t]}, e^{s[63]-s[t]}
struct Decays {
    float hi[kQ], lo[kQ], step[kQ], from[kQ], to[kQ];
};

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// by one wave for one chunk; `raw`: this lane's dt (with bias), `alive`: whether its token is within the row
__device__ __forceinline__ void put_decays(Decays& o, float raw, bool alive, bool plus, float A) {
    const int lane = threadIdx.x & 63;
    const float d = !alive ? 0.f : plus ? softplus(raw) : raw;
    float hi, lo;
    chunk_decay(d, A, hi, lo);
    const float eh = __shfl(hi, 63, 64), el = __shfl(lo, 63, 64);
    o.hi[lane] = hi, o.lo[lane] = lo, o.step[lane] = d, o.from[lane] = exp2_fast(hi), o.to[lane] = exp2_fast((eh - hi) + (el - lo));
}

// blocks that follow each other share inputs (heads of a group): hand each XCD a contiguous part of them (workgroup i runs on XCD i % 8)
__device__ __forceinline__ unsigned xcd_block(unsigned i, unsigned n) {
    const unsigned q = n >> 3, r = n & 7, x = i & 7, k = i >> 3;
    return x * q + (x < r ? x : r) + k;
}

// ---- arguments and host side (ssm_scan.hip) --------------------------------------------------------------------------------------------------------------
struct ScanArgs {
    const void *x, *B, *C;
    long long x_row, x_tok, b_row, b_tok, c_row, c_tok;
    Steps dt;
    const float *A, *D, *state;
    const int* lengths;
    int rows, L, H, P, G, N;
    int segs, seg_chunks, chunks;  // segments per row, chunks per segment and per row
    int fast_x, fast_b, fast_c;
};

__device__ __forceinline__ int row_length(const int* lengths, int b, int L) {
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : n < L ? n : L;
}

struct WalkOut {
    const float* starts;  // [row][head][segment][PP][NP], or none: segments start from zero
    float *ends, *decays;
    float* tiles;         // [row][chunk][head][PP * NP]
    float* last;          // [row][head][P][N]
    int backwards;
};


template <int PP> struct Waves {
    static constexpr int kWaves = PP / 16 < 4 ? PP / 16 : 4, kThreads = 64 * kWaves, kTiles = PP / 16 / kWaves;  // 16-wide slices of P per wave
};

// P and N are padded to 32, 64 or 128 in LDS and registers (the padding is zero, in memory there is none)
inline int padded(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }
inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline bool scan_sizes(int B, int L, int H, int P, int G, int N) {
    return B > 0 && L > 0 && L <= (1 << 30) && H > 0 && P > 0 && P <= 128 && G > 0 && H % G == 0 && N > 0 && N <= 128 && (long long)B * H <= (1 << 24);
}

void scan_cut(ScanArgs& a);
int scan_starts(const ScanArgs& a0, const ScanArgs& a1, const float* state1, float* ws, int both, int type, hipStream_t st);
int scan_walks(const ScanArgs& a0, const WalkOut& o0, const ScanArgs& a1, const WalkOut& o1, int both, int type, hipStream_t st);

inline ScanArgs scan_args(const void* x, long long x_row, long long x_tok, const Steps& dt, const float* A, const void* B, long long b_row, long long b_tok,
                          const void* C, long long c_row, long long c_tok, const float* D, const float* state, const int* lengths, int rows, int L, int H, int P,
                          int G, int N, int type) {
    ScanArgs a{x, B, C, x_row, x_tok, b_row, b_tok, c_row, c_tok, dt, A, D, state, lengths, rows, L, H, P, G, N, 1, 0, 0, 0, 0, 0};
    const int v = type == 0 ? 4 : 8;  // values in 16 bytes; 64 tokens must lie within 2^31 bytes of each other
    auto fast = [&](const void* p, int width, long long row, long long tok) {
        return width % v == 0 && row % v == 0 && tok % v == 0 && tok >= 0 && tok < (1ll << 23) && on16(p);
    };
    a.fast_x = fast(x, P, x_row, x_tok), a.fast_b = fast(B, N, b_row, b_tok), a.fast_c = fast(C, N, c_row, c_tok);
    scan_cut(a);
    return a;
}

#define RTFS_SSM_PP(T, NP, P, F, ARGS)         \
    do {                                       \
        if ((P) <= 32) return F<T, NP, 32> ARGS; \
        if ((P) <= 64) return F<T, NP, 64> ARGS; \
        return F<T, NP, 128> ARGS;             \
    } while (0)
#define RTFS_SSM_NP(T, N, P, F, ARGS)                      \
    do {                                                   \
        if ((N) <= 32) RTFS_SSM_PP(T, 32, P, F, ARGS);     \
        else if ((N) <= 64) RTFS_SSM_PP(T, 64, P, F, ARGS); \
        else RTFS_SSM_PP(T, 128, P, F, ARGS);              \
    } while (0)
#define RTFS_SSM_DISPATCH(type, N, P, F, ARGS)         \
    do {                                               \
        if ((type) == 0) RTFS_SSM_NP(float, N, P, F, ARGS); \
        else RTFS_SSM_NP(__bf16, N, P, F, ARGS);       \
    } while (0)

}  // namespace ssm
}  // namespace rtfs
