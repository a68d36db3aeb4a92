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
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// ---- fragments ------------------------------------------------------------------------------------------------------------------------------------------
// One fragment is a 16 x 32 operand of D[16x16] += A[16x32] B[32x16]: lane l holds 8 values of row (A) or column (B) l & 15; which 8 of the 32 products it
// holds is free as long as A and B agree.  Here, with g = l >> 4: k = 4 g + j and 16 + 4 g + j (j < 4), which is how two accumulator tiles lie in registers
// (lane l: column l & 15, rows 4 g + i) - an accumulator becomes an operand without leaving its lane.
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
template <typename T> __device__ __forceinline__ Frag<T> frag_of(f32x4 a, f32x4 b);
template <> __device__ __forceinline__ Frag<float> frag_of<float>(f32x4 a, f32x4 b) { return {a, b}; }
template <> __device__ __forceinline__ Frag<__bf16> frag_of<__bf16>(f32x4 a, f32x4 b) {
    return {__builtin_shufflevector(__builtin_convertvector(a, bf16x4), __builtin_convertvector(b, bf16x4), 0, 1, 2, 3, 4, 5, 6, 7)};
}
// An fp32 operand as the sum of three bf16, 8 bits of its 24-bit mantissa each and so exact: states, what builds them, and the sums that the gradients of dt and A
// are differences of keep fp32's precision for bf16 tensors too.  fp32 operands are themselves.
template <typename T> struct Split {
    static constexpr int kTerms = 3;
    Frag<T> hi, mid, lo;
    __device__ __forceinline__ const Frag<T>& part(int i) const { return i == 0 ? hi : i == 1 ? mid : lo; }
};
template <> struct Split<float> {
    static constexpr int kTerms = 1;
    Frag<float> hi;
    __device__ __forceinline__ const Frag<float>& part(int) const { return hi; }
};
__device__ __forceinline__ void split(f32x4 a, f32x4 b, Split<float>& s) { s.hi = {a, b}; }
// the upper halves of eight fp32 as bf16 (cut off, not rounded); what they leave stays in a and b
__device__ __forceinline__ Frag<__bf16> take_upper(f32x4& a, f32x4& b) {
    const u32x4 x = __builtin_bit_cast(u32x4, a), y = __builtin_bit_cast(u32x4, b);
    const u32x4 v = {__builtin_amdgcn_perm(x[1], x[0], 0x07060302u), __builtin_amdgcn_perm(x[3], x[2], 0x07060302u),
                     __builtin_amdgcn_perm(y[1], y[0], 0x07060302u), __builtin_amdgcn_perm(y[3], y[2], 0x07060302u)};
    a -= __builtin_bit_cast(f32x4, x & 0xffff0000u);
    b -= __builtin_bit_cast(f32x4, y & 0xffff0000u);
    return {__builtin_bit_cast(bf16x8, v)};
}
__device__ __forceinline__ void split(f32x4 a, f32x4 b, Split<__bf16>& s) { s.hi = take_upper(a, b), s.mid = take_upper(a, b), s.lo = take_upper(a, b); }
__device__ __forceinline__ f32x4 mma(const Frag<float>& x, const Split<float>& y, f32x4 c) { return mma(x, y.hi, c); }
__device__ __forceinline__ f32x4 mma(const Frag<__bf16>& x, const Split<__bf16>& y, f32x4 c) { return mma(x, y.hi, mma(x, y.mid, mma(x, y.lo, c))); }

__device__ __forceinline__ void widen(const Frag<float>& f, f32x4& a, f32x4& b) { a = f.a, b = f.b; }
__device__ __forceinline__ void widen(const Frag<__bf16>& f, f32x4& a, f32x4& b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (float)f.v[j], b[j] = (float)f.v[4 + j];
}

// ---- tiles in LDS -----------------------------------------------------------------------------------------------------------------------------------------
// ROWS x COLS values, read two ways as operands: 4 + 4 neighbours of a row (products over values: row()), and 4 + 4 rows of a column (products over tokens:
// down()).  fp32 takes down() one value at a time, as many bytes per cycle; rows are 16 bytes apart from a multiple of all banks.  bf16 takes it with the
// transposing read ds_read_b64_tr_b16 (16 lanes fetch four rows of 16 values, each lane gets one column of them), so no tile is stored twice.  Its rows have no
// padding; instead the 8-byte granules of a row are permuted by an exclusive or with a code of the row that sends the 16 rows of a row() read and the four
// rows x four granules of a down() read to 16 different pairs of banks (a tile of 16 columns is only read down(): it needs none).
template <typename T> struct Vec8;
template <> struct Vec8<float> { f32x4 a, b; };
template <> struct Vec8<__bf16> { bf16x8 v; };
// Where a lane reads, in values from the start of a tile of COLS columns; formed once, all else is a constant added to it.
template <typename T, int COLS> struct Lanes;
template <int COLS> struct Lanes<float, COLS> {
    static constexpr int kPitch = COLS + 4;
    int row, down;
    __device__ __forceinline__ Lanes() {
        const int lane = threadIdx.x & 63, lc = lane & 15, g = lane >> 4;
        row = lc * kPitch + 4 * g, down = 4 * g * kPitch + lc;
    }
};
template <int COLS> struct Lanes<__bf16, COLS> {
    // Granules c / 4 of a row r lie at (c / 4) ^ code(r): 16 (COLS = 32: 8, 16: 4) of them permuted, the codes chosen so that ...
    __device__ __forceinline__ static int code(int r) {
        return COLS >= 64 ? (r & 3) << 2 | ((r >> 2) & 3) : COLS == 32 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : 0;
    }
    // ... a constant granule 4 v in front of a lane's own is an exclusive or with it: one offset per v, and the rest of the constant is added
    static constexpr int kOffsets = COLS >= 64 ? 4 : COLS / 16;
    int row[kOffsets], down[kOffsets];
    __device__ __forceinline__ Lanes() {
        const int lane = threadIdx.x & 63, lc = lane & 15, g = lane >> 4, r = 4 * g + (lc >> 2);
#pragma unroll
        for (int v = 0; v < kOffsets; ++v) {
            row[v] = lc * COLS + ((g ^ code(lc) ^ v << 2) << 2);
            down[v] = r * COLS + (((lc & 3) ^ code(r) ^ v << 2) << 2);
        }
    }
};

template <typename T, int ROWS, int COLS> struct Tile;

template <int ROWS, int COLS> struct Tile<float, ROWS, COLS> {
    typedef Lanes<float, COLS> Lane;
    static constexpr int kPitch = Lane::kPitch, kBytes = ROWS * kPitch * 4;
    float v[ROWS * kPitch];
    __device__ __forceinline__ void put8(int r, int c, const Vec8<float>& x) {
        *reinterpret_cast<f32x4*>(v + r * kPitch + c) = x.a;
        *reinterpret_cast<f32x4*>(v + r * kPitch + c + 4) = x.b;
    }
    __device__ __forceinline__ void put4(int r, int c, f32x4 x) { *reinterpret_cast<f32x4*>(v + r * kPitch + c) = x; }
    __device__ __forceinline__ void put(int r, int c, float x) { v[r * kPitch + c] = x; }
    __device__ __forceinline__ float get(int r, int c) const { return v[r * kPitch + c]; }
    // r, c: multiples of 16.  Lane l: row r + (l & 15), values c + 4 g .. and c + 16 + 4 g ..
    __device__ __forceinline__ Frag<float> row(const Lane& l, int r, int c) const {
        const float* p = v + l.row + r * kPitch + c;
        return {*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + 16)};
    }
    __device__ __forceinline__ Frag<float> down_any(int r, int c) const { return down(Lane(), r, c); }
    // lane l: column c + (l & 15), rows r + 4 g .. and r + 16 + 4 g ..
    __device__ __forceinline__ Frag<float> down(const Lane& l, int r, int c) const {
        const float* p = v + l.down + r * kPitch + c;
        Frag<float> f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f.a[j] = p[j * kPitch], f.b[j] = p[(16 + j) * kPitch];
        return f;
    }
};

template <int ROWS, int COLS> struct Tile<__bf16, ROWS, COLS> {
    typedef Lanes<__bf16, COLS> Lane;
    static constexpr int kBytes = ROWS * COLS * 2;
    __bf16 v[ROWS * COLS];
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    __device__ __forceinline__ static int at(int r, int c) { return r * COLS + ((c >> 2 ^ Lane::code(r)) << 2 | (c & 3)); }
    __device__ __forceinline__ void put8(int r, int c, const Vec8<__bf16>& x) {
        *reinterpret_cast<bf16x4*>(v + at(r, c)) = __builtin_shufflevector(x.v, x.v, 0, 1, 2, 3);
        *reinterpret_cast<bf16x4*>(v + at(r, c + 4)) = __builtin_shufflevector(x.v, x.v, 4, 5, 6, 7);
    }
    __device__ __forceinline__ void put4(int r, int c, f32x4 x) { *reinterpret_cast<bf16x4*>(v + at(r, c)) = __builtin_convertvector(x, bf16x4); }
    __device__ __forceinline__ void put(int r, int c, float x) { v[at(r, c)] = (__bf16)x; }
    __device__ __forceinline__ float get(int r, int c) const { return (float)v[at(r, c)]; }
    __device__ __forceinline__ Frag<__bf16> row(const Lane& l, int r, int c) const {
        constexpr int m = Lane::kOffsets - 1;
        const __bf16* p = v + r * COLS + (c >> 6 << 6);
        const bf16x4 a = *reinterpret_cast<const bf16x4*>(p + l.row[c >> 4 & m]), b = *reinterpret_cast<const bf16x4*>(p + l.row[(c + 16) >> 4 & m]);
        return {__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7)};
    }
    __device__ __forceinline__ Frag<__bf16> down(const Lane& l, int r, int c) const {
        return down_from(v + r * COLS + (c >> 6 << 6) + l.down[c >> 4 & (Lane::kOffsets - 1)]);
    }
    // the same where c is not known to the compiler
    __device__ __forceinline__ Frag<__bf16> down_any(int r, int c) const {
        const int lane = threadIdx.x & 63;
        return down_from(v + at(r + 4 * (lane >> 4) + (lane >> 2 & 3), c + 4 * (lane & 3)));
    }
    __device__ __forceinline__ static Frag<__bf16> down_from(const __bf16* p) {
        typedef __attribute__((address_space(3))) s16x4* lds;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + 16 * COLS));
        return {__builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7))};
    }
};

// 8 values at byte offset `at`, the first `n` of them; bounds are below 2^31, so the offset of a value that is not wanted is set past them and reads as zero
constexpr unsigned kNowhere = 0x80000000u;
__device__ __forceinline__ void load8(Vec8<__bf16>& v, __amdgpu_buffer_rsrc_t r, unsigned at, int n) {
    v.v = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, n > 0 ? at : kNowhere, 0, 0));
}
__device__ __forceinline__ void load8(Vec8<float>& v, __amdgpu_buffer_rsrc_t r, unsigned at, int n) {
    v.a = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, n > 0 ? at : kNowhere, 0, 0));
    v.b = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, n > 4 ? at + 16 : kNowhere, 0, 0));
}
// 16 bytes at any address, also where fewer values than that are left in a row (`n`, of rows of at least 16 bytes): the 16 bytes that end with the row then, moved
// down - so no byte behind a row's last value is asked for
__device__ __forceinline__ u32x4 load16_ending(__amdgpu_buffer_rsrc_t r, unsigned at, int missing_words, bool any) {
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(r, any ? at - 4 * missing_words : kNowhere, 0, 0);
    const bool two = missing_words & 2, one = missing_words & 1;
    const unsigned a = two ? v[2] : v[0], b = two ? v[3] : v[1], c = two ? 0u : v[2], d = two ? 0u : v[3];
    return u32x4{one ? b : a, one ? c : b, one ? d : c, one ? 0u : d};
}
__device__ __forceinline__ void load8_anywhere(Vec8<__bf16>& v, __amdgpu_buffer_rsrc_t r, unsigned at, int n) {
    const int missing = n >= 8 || n <= 0 ? 0 : 8 - n;
    const u32x4 x = load16_ending(r, at - 2 * (missing & 1), missing >> 1, n > 0);
    const unsigned half = missing & 1 ? 16u : 0u;
    v.v = __builtin_bit_cast(bf16x8, u32x4{__builtin_amdgcn_alignbit(x[1], x[0], half), __builtin_amdgcn_alignbit(x[2], x[1], half),
                                           __builtin_amdgcn_alignbit(x[3], x[2], half), x[3] >> half});
}
__device__ __forceinline__ void load8_anywhere(Vec8<float>& v, __amdgpu_buffer_rsrc_t r, unsigned at, int n) {
    v.a = __builtin_bit_cast(f32x4, load16_ending(r, at, n >= 4 || n <= 0 ? 0 : 4 - n, n > 0));
    v.b = __builtin_bit_cast(f32x4, load16_ending(r, at + 16, n >= 8 || n <= 4 ? 0 : 8 - n, n > 4));
}
__device__ __forceinline__ void load8_singly(Vec8<__bf16>& v, __amdgpu_buffer_rsrc_t r, unsigned at, int n) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v.v[j] = __builtin_bit_cast(__bf16, __builtin_amdgcn_raw_buffer_load_b16(r, n > j ? at + 2 * j : kNowhere, 0, 0));
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void load8_singly(Vec8<float>& v, __amdgpu_buffer_rsrc_t r, unsigned at, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v.a[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, n > j ? at + 4 * j : kNowhere, 0, 0));
        v.b[j] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, n > 4 + j ? at + 16 + 4 * j : kNowhere, 0, 0));
    }
    __builtin_amdgcn_sched_barrier(0);
}

// 64 tokens of up to COLS values on their way from memory to a Tile, 8 values at a time, by THREADS threads; what lies past `rows` tokens or `cols` values is
// zero and never read (a padded batch may hold anything there).  Buffer loads throughout: their bounds check supplies the zeros without a branch, and code
// without branches lets the loads stay in flight until put() - a tile is asked for ahead of the work on the one before.  `how` the rows lie:
enum { kAligned = 0, kAnywhere = 1, kShort = 2 };  // on 16 bytes, `cols` a multiple of them; rows of at least 16 bytes; shorter ones (and what a slice leaves of one), value by value
template <typename T, int COLS, int THREADS>
struct Load {
    static constexpr int kVecs = COLS / 8, kUnits = kQ * kVecs, kPer = (kUnits + THREADS - 1) / THREADS;
    Vec8<T> r[kPer];

    __device__ __forceinline__ void ask(unsigned thread, const T* src, long long pitch, int rows, int cols, int how) {
        // formed anew at every call: hoisted out of the chunk loop, the addresses of the value-by-value path alone take a hundred registers
        asm volatile("" : "+v"(thread));
        // without a token the bound is 0: nothing is read (below 0 it would be no bound at all)
        const int bytes = rows > 0 ? (int)(((rows - 1) * pitch + cols) * (long long)sizeof(T)) : 0;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(src), 0, bytes, 0x00027000);
        const unsigned step = (unsigned)pitch * sizeof(T);
        auto all = [&](auto load) {
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const unsigned u = thread + k * THREADS, c = u % kVecs * 8, at = u / kVecs * step + c * (unsigned)sizeof(T);
                load(r[k], at, kUnits % THREADS == 0 || u < kUnits ? cols - (int)c : 0);
            }
        };
        if (how == kAligned) all([&](Vec8<T>& v, unsigned at, int n) { load8(v, rsrc, at, n); });
        else if (how == kAnywhere && cols * (int)sizeof(T) >= 16) all([&](Vec8<T>& v, unsigned at, int n) { load8_anywhere(v, rsrc, at, n); });
        else all([&](Vec8<T>& v, unsigned at, int n) { load8_singly(v, rsrc, at, n); });
    }
    __device__ __forceinline__ void put(unsigned thread, Tile<T, kQ, COLS>& tile) const {
        asm volatile("" : "+v"(thread));
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const unsigned u = thread + k * THREADS;
            if (kUnits % THREADS == 0 || u < kUnits) tile.put8(u / kVecs, u % kVecs * 8, r[k]);
        }
    }
};

// this wave's index, known to the compiler to be the same in all its lanes
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---- decays ---------------------------------------------------------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f;

// log(1 + e^v): e^v with the rounding of v log2 e made good, and the logarithm of 1 + x as log(u) x / (u - 1) with u = 1 + x rounded - where x is small the
// quotient gives back what the sum lost
__device__ __forceinline__ float softplus(float v) {
    const float m = -fminf(fabsf(v), 200.f), t = m * kLog2e, rest = fmaf(m, kLog2e, -t) + m * 1.925963033500e-8f;  // log2 e = kLog2e + 1.926e-8
    const float x = __builtin_amdgcn_exp2f(t) * fmaf(rest, 0.693147181f, 1.f), u = 1.f + x, d = u - 1.f;
    const float l = d == 0.f ? x : __builtin_amdgcn_logf(u) * 0.693147181f * (x * __builtin_amdgcn_rcpf(d));
    return v != v ? v : fmaxf(v, 0.f) + l;
}

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

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
    const long long bits = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)bits, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(bits >> 32), CTRL, ROWS, 0xf, false);
    return v + __builtin_bit_cast(double, (long long)(unsigned)lo | (long long)hi << 32);
}
// Sums over the tokens up to and including this lane's, in fp64: the differences s[t] - s[j] are what counts, and behind a strong decay both are large.
// Shifts inside the rows of 16 lanes, then the rows' last lanes handed on; lanes a step does not reach add 0.
__device__ __forceinline__ double running_sum(double v) {
    v = dpp_add<0x111, 0xf>(v);  // row_shr:1
    v = dpp_add<0x112, 0xf>(v);  // row_shr:2
    v = dpp_add<0x114, 0xf>(v);  // row_shr:4
    v = dpp_add<0x118, 0xf>(v);  // row_shr:8
    v = dpp_add<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    return dpp_add<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
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
    int width, slices, quads;      // columns of P per wave, waves per head, workgroups (four waves) per group of heads
    int how_x, how_b, how_c;  // how their rows lie (Load)
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


// P and N are padded to 32, 64 or 128 in LDS and registers (the padding is zero, in memory there is none)
__host__ __device__ constexpr int padded(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : 128; }
inline bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline bool scan_sizes(int B, int L, int H, int P, int G, int N) {
    return B > 0 && L > 0 && L <= (1 << 30) && H > 0 && P > 0 && P <= 128 && G > 0 && H % G == 0 && N > 0 && N <= 128 && (long long)B * H <= (1 << 24);
}

// 64 tokens must lie within 2^31 bytes of each other: buffer offsets
inline bool scan_pitch(long long tok) { return tok >= 0 && tok < (1ll << 23); }

void scan_cut(ScanArgs& a);
int scan_starts(const ScanArgs& a0, const ScanArgs& a1, const float* state1, float* ws, int both, int type, hipStream_t st);
int scan_walks(const ScanArgs& a0, const WalkOut& o0, const ScanArgs& a1, const WalkOut& o1, int both, int type, hipStream_t st);

inline ScanArgs scan_args(const void* x, long long x_row, long long x_tok, const Steps& dt, const float* A, const void* B, long long b_row, long long b_tok,
                          const void* C, long long c_row, long long c_tok, const float* D, const float* state, const int* lengths, int rows, int L, int H, int P,
                          int G, int N, int type) {
    ScanArgs a{x, B, C, x_row, x_tok, b_row, b_tok, c_row, c_tok, dt, A, D, state, lengths, rows, L, H, P, G, N, 1, 0, 0, 0, 0, 0, 0, 0, 0};
    const int v = type == 0 ? 4 : 8;  // values in 16 bytes
    auto how = [&](const void* p, int width, long long row, long long tok) {
        return width % v == 0 && row % v == 0 && tok % v == 0 && on16(p) ? kAligned : width >= v ? kAnywhere : kShort;
    };
    a.how_x = how(x, P, x_row, x_tok), a.how_b = how(B, N, b_row, b_tok), a.how_c = how(C, N, c_row, c_tok);
    scan_cut(a);
    return a;
}

// type and sizes -> template; W is the width of a wave's slice of P (scan, walks; at most LAST where N > 64) or the padded P (gradients), from FIRST on
#define RTFS_SSM_W(T, NP, FIRST, LAST, W, F, ARGS)                                              \
    do {                                                                                        \
        if ((W) <= (FIRST)) return F<T, NP, (FIRST)> ARGS;                                      \
        if ((W) <= 2 * (FIRST) || 2 * (FIRST) == (LAST)) return F<T, NP, 2 * (FIRST)> ARGS;     \
        return F<T, NP, 2 * (FIRST) == (LAST) ? (LAST) : 4 * (FIRST)> ARGS;                     \
    } while (0)
#define RTFS_SSM_NP(T, N, FIRST, LAST, W, F, ARGS)                              \
    do {                                                                        \
        if ((N) <= 32) RTFS_SSM_W(T, 32, FIRST, 4 * (FIRST), W, F, ARGS);       \
        else if ((N) <= 64) RTFS_SSM_W(T, 64, FIRST, 4 * (FIRST), W, F, ARGS);  \
        else RTFS_SSM_W(T, 128, FIRST, LAST, W, F, ARGS);                       \
    } while (0)
#define RTFS_SSM_DISPATCH(type, N, FIRST, LAST, W, F, ARGS)              \
    do {                                                                 \
        if ((type) == 0) RTFS_SSM_NP(float, N, FIRST, LAST, W, F, ARGS); \
        else RTFS_SSM_NP(__bf16, N, FIRST, LAST, W, F, ARGS);            \
    } while (0)

}  // namespace ssm
}  // namespace rtfs
