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
// holds is free as long as A and B agree.  With g = l >> 4, two accumulator tiles (lane l: column l & 15, rows 4 g + i) become an operand without leaving their
// lane, of the products 4 g + j and 16 + 4 g + j (j < 4) of their 32 rows - or of 8 g + j and 8 g + 4 + j, if row 4 g + i of the pair's first tile stands for
// value 8 g + i and that of its second for 8 g + 4 + i.  The latter is how tiles over N lie (swapped()), so that rows of B and C are read 16 bytes at a time.
// fp32 goes through v_mfma_f32_16x16x4_f32 (exact products, one value per lane and step), bf16 through one v_mfma_f32_16x16x32_bf16.  (fp32 as three bf16 terms
// and six products takes 96 cycles for 256, but 52 vector instructions to split an operand: 2048 rows of 125 tokens, 4 heads of 32, N = 32, forward and gradients
// 588 us against 589, and an infinity becomes a NaN.)
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
// what rounding to bf16 leaves of them
__device__ __forceinline__ f32x4 rest_of(f32x4 a) { return a - __builtin_convertvector(__builtin_convertvector(a, bf16x4), f32x4); }
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
__device__ __forceinline__ f32x4 mma(const Split<float>& x, const Frag<float>& y, f32x4 c) { return mma(x.hi, y, c); }
__device__ __forceinline__ f32x4 mma(const Split<__bf16>& x, const Frag<__bf16>& y, f32x4 c) { return mma(x.hi, y, mma(x.mid, y, mma(x.lo, y, c))); }

__device__ __forceinline__ void widen(const Frag<float>& f, f32x4& a, f32x4& b) { a = f.a, b = f.b; }
__device__ __forceinline__ void widen(const Frag<__bf16>& f, f32x4& a, f32x4& b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (float)f.v[j], b[j] = (float)f.v[4 + j];
}

// the value of N that place i (0 .. 15) of tile t stands for
__device__ __forceinline__ int swapped(int t, int i) { return 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3); }

// ---- tiles in LDS -----------------------------------------------------------------------------------------------------------------------------------------
// ROWS x COLS values, read two ways as operands: 8 values of a row (products over values: row()), and 4 + 4 rows of a column (products over tokens: down()).
// Three KINDs, by what their accumulator tiles are to be:
//   kSwapped  B and C: row() gives values 8 g .. 8 g + 7; lane i of a down() tile gets column swapped(t, i)
//   kInOrder  x and dy of the gradients, scores: row() gives values 4 g .. and 16 + 4 g ..; lane i of a down() tile gets column 16 t + i
//   kDownOnly x of the scan, states: down() as kInOrder, no row()
// fp32 takes down() one value at a time, as many bytes per cycle; rows are 16 bytes apart from a multiple of all banks.  bf16 takes it with the transposing
// read ds_read_b64_tr_b16 (16 lanes fetch four rows of 16 values, each lane gets one column of them), so no tile is stored twice.  Its rows have no padding;
// their 16-byte chunks are permuted by an exclusive or with a code of the row instead: the eight rows of a phase of row() and the four rows of down() meet
// different banks (kSwapped's down(): twice each, it takes one half of every chunk).  kInOrder stores granules of four so that the 16 bytes row() reads are the
// right ones.
enum Kind { kSwapped, kInOrder, kDownOnly };

template <typename T> struct Vec8;
template <> struct Vec8<float> { f32x4 a, b; };
template <> struct Vec8<__bf16> { bf16x8 v; };

// Where a lane reads, in values from the start of a tile of COLS columns; formed once, all else is a constant added to it.
template <typename T, int COLS, Kind KIND> struct Lanes;
template <int COLS, Kind KIND> struct Lanes<float, COLS, KIND> {
    static constexpr int kPitch = COLS + 4;
    int row, down;
    __device__ __forceinline__ Lanes() {
        const int lane = threadIdx.x & 63, lc = lane & 15, g = lane >> 4;
        row = lc * kPitch + (KIND == kSwapped ? 8 * g : 4 * g), down = 4 * g * kPitch + (KIND == kSwapped ? swapped(0, lc) : lc);
    }
};
template <int COLS, Kind KIND> struct Lanes<__bf16, COLS, KIND> {
    // chunk c of row r lies at c ^ code(r); 128 bytes of banks hold one row of 64 values, two of 32, four of 16
    __device__ __forceinline__ static int code(int r) { return COLS >= 64 ? (r & 1) << 2 | (r & 2) | ((r >> 2) & 1) : COLS == 32 ? (r & 2) | ((r >> 2) & 1) : 0; }
    // a constant chunk in front of a lane's own is an exclusive or with it where it is among the permuted ones: one offset each, the rest is added
    static constexpr int kRow = COLS >= 64 ? 2 : 1, kDown = KIND != kDownOnly ? kRow : COLS >= 64 ? 4 : COLS / 16;
    int row[kRow], down[kDown];
    __device__ __forceinline__ Lanes() {
        const int lane = threadIdx.x & 63, lc = lane & 15, g = lane >> 4, r = 4 * g + (lc >> 2), q = lc & 3;
#pragma unroll
        for (int v = 0; v < kRow; ++v) row[v] = lc * COLS + ((g ^ code(lc) ^ v << 2) << 3);
#pragma unroll
        for (int v = 0; v < kDown; ++v)
            down[v] = r * COLS + (KIND != kDownOnly ? (q ^ code(r) ^ v << 2) << 3 : ((q >> 1) ^ code(r) ^ v << 1) << 3 | (q & 1) << 2);
    }
};

template <typename T, int ROWS, int COLS, Kind KIND> struct Tile;

template <int ROWS, int COLS, Kind KIND> struct Tile<float, ROWS, COLS, KIND> {
    typedef Lanes<float, COLS, KIND> Lane;
    static constexpr int kPitch = Lane::kPitch, kBytes = ROWS * kPitch * 4;
    float v[ROWS * kPitch];
    // where 8 neighbours of a row go; rows 8 apart are 8 * kPitch apart
    struct Place {
        int at;
        __device__ __forceinline__ Place(int r, int c) : at(r * kPitch + c) {}
    };
    __device__ __forceinline__ void put8(const Place& p, int rows, const Vec8<float>& x) {
        *reinterpret_cast<f32x4*>(v + p.at + rows * kPitch) = x.a;
        *reinterpret_cast<f32x4*>(v + p.at + rows * kPitch + 4) = x.b;
    }
    __device__ __forceinline__ void put4(int r, int c, f32x4 x) { *reinterpret_cast<f32x4*>(v + r * kPitch + c) = x; }
    __device__ __forceinline__ f32x4 get4(int r, int c) const { return *reinterpret_cast<const f32x4*>(v + r * kPitch + c); }
    __device__ __forceinline__ void put(int r, int c, float x) { v[r * kPitch + c] = x; }
    // lane l: row r + (l & 15), values from c (a multiple of 32) on
    __device__ __forceinline__ Frag<float> row(const Lane& l, int r, int c) const {
        const float* p = v + l.row + r * kPitch + c;
        return {*reinterpret_cast<const f32x4*>(p), *reinterpret_cast<const f32x4*>(p + (KIND == kSwapped ? 4 : 16))};
    }
    __device__ __forceinline__ Frag<float> row_any(const Lane& l, int r, int c) const { return row(l, r, c); }  // c not known to the compiler
    // lane l: place l & 15 of column tile t, rows r + 4 g .. and r + 16 + 4 g ..
    __device__ __forceinline__ Frag<float> down(const Lane& l, int r, int t) const {
        const float* p = v + l.down + r * kPitch + (KIND == kSwapped ? swapped(t, 0) : 16 * t);
        Frag<float> f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f.a[j] = p[j * kPitch], f.b[j] = p[(16 + j) * kPitch];
        return f;
    }
    __device__ __forceinline__ Frag<float> down_any(int r, int t) const { return down(Lane(), r, t); }
};

template <int ROWS, int COLS, Kind KIND> struct Tile<__bf16, ROWS, COLS, KIND> {
    typedef Lanes<__bf16, COLS, KIND> Lane;
    static constexpr int kBytes = ROWS * COLS * 2;
    __bf16 v[ROWS * COLS];
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    // four neighbours from column c (a multiple of 4) on; granule 4 h + g of eight is stored as 2 g + h where KIND is kInOrder
    __device__ __forceinline__ static int at(int r, int c) {
        const int q = c >> 2, s = KIND == kInOrder ? (q & ~7) | (q & 3) << 1 | ((q >> 2) & 1) : q;
        return r * COLS + ((s >> 1 ^ Lane::code(r)) << 3 | (s & 1) << 2 | (c & 3));
    }
    struct Place {
        int at0, at1;
        __device__ __forceinline__ Place(int r, int c) : at0(at(r, c)), at1(KIND == kInOrder ? at(r, c + 4) : 0) {}
    };
    __device__ __forceinline__ void put8(const Place& p, int rows, const Vec8<__bf16>& x) {
        if (KIND == kInOrder) {
            *reinterpret_cast<bf16x4*>(v + p.at0 + rows * COLS) = __builtin_shufflevector(x.v, x.v, 0, 1, 2, 3);
            *reinterpret_cast<bf16x4*>(v + p.at1 + rows * COLS) = __builtin_shufflevector(x.v, x.v, 4, 5, 6, 7);
        } else {
            *reinterpret_cast<bf16x8*>(v + p.at0 + rows * COLS) = x.v;
        }
    }
    __device__ __forceinline__ void put4(int r, int c, f32x4 x) { *reinterpret_cast<bf16x4*>(v + at(r, c)) = __builtin_convertvector(x, bf16x4); }
    __device__ __forceinline__ f32x4 get4(int r, int c) const { return __builtin_convertvector(*reinterpret_cast<const bf16x4*>(v + at(r, c)), f32x4); }
    __device__ __forceinline__ void put(int r, int c, float x) { v[at(r, c)] = (__bf16)x; }
    __device__ __forceinline__ Frag<__bf16> row(const Lane& l, int r, int c) const {
        return {*reinterpret_cast<const bf16x8*>(v + r * COLS + (c >> 6 << 6) + l.row[c >> 5 & (Lane::kRow - 1)])};
    }
    __device__ __forceinline__ Frag<__bf16> row_any(const Lane& l, int r, int c) const {
        return {*reinterpret_cast<const bf16x8*>(v + r * COLS + (c >> 6 << 6) + (c >> 5 & (Lane::kRow - 1) ? l.row[Lane::kRow - 1] : l.row[0]))};
    }
    __device__ __forceinline__ Frag<__bf16> down(const Lane& l, int r, int t) const {
        if (KIND == kDownOnly) return down_from(v + r * COLS + (t >> 2 << 6) + l.down[t & (Lane::kDown - 1)]);
        return down_from(v + r * COLS + (t >> 2 << 6) + 4 * (t & 1) + l.down[t >> 1 & (Lane::kDown - 1)]);
    }
    __device__ __forceinline__ Frag<__bf16> down_any(int r, int t) const {
        const int lane = threadIdx.x & 63, m = r + 4 * (lane >> 4) + (lane >> 2 & 3), q = lane & 3;
        return down_from(v + at(m, KIND == kSwapped ? swapped(t, 4 * q) : 16 * t + 4 * q));
    }
    __device__ __forceinline__ static Frag<__bf16> down_from(const __bf16* p) {
        typedef __attribute__((address_space(3))) s16x4* lds;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + 16 * COLS));
        return {__builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7))};
    }
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
// v += 0 x of all x of a Vec8
__device__ __forceinline__ void times_zero(const Vec8<float>& x, float& v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v = fmaf(x.a[j], 0.f, v), v = fmaf(x.b[j], 0.f, v);
}
__device__ __forceinline__ void times_zero(const Vec8<__bf16>& x, float& v) {
    const bf16x2 zero = {(__bf16)0.f, (__bf16)0.f};
#pragma unroll
    for (int j = 0; j < 8; j += 2) v = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x.v[j], x.v[j + 1]}, zero, v, false);
}
__device__ __forceinline__ float value(const Vec8<float>& x, int j) { return j < 4 ? x.a[j] : x.b[j - 4]; }
__device__ __forceinline__ float value(const Vec8<__bf16>& x, int j) { return (float)x.v[j]; }
__device__ __forceinline__ void clear(Vec8<float>& x, int j) {
    if (j < 4) x.a[j] = 0.f;
    else x.b[j - 4] = 0.f;
}
__device__ __forceinline__ void clear(Vec8<__bf16>& x, int j) { x.v[j] = (__bf16)0.f; }

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
// ANEW: offsets of aligned rows are formed at every call too, a dozen registers fewer over the chunk loop (prompts in bf16, which spill otherwise: 32768 tokens, 32 heads
// of 64, N = 128: 290 us, 274 with it; fp32 gradients of 2048 rows of 125 tokens, 4 heads of 32, which do not: 565 us, 556 without).
template <typename T, int COLS, int THREADS, bool ANEW = false>
struct Load {
    static constexpr int kVecs = COLS / 8, kUnits = kQ * kVecs, kPer = (kUnits + THREADS - 1) / THREADS;
    Vec8<T> r[kPer];

    __device__ __forceinline__ void ask(unsigned thread, const T* src, long long pitch, int rows, int cols, int how) {
        // without a token the bound is 0: nothing is read (below 0 it would be no bound at all)
        const int bytes = rows > 0 ? (int)(((rows - 1) * pitch + cols) * (long long)sizeof(T)) : 0;
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(src), 0, bytes, 0x00027000);
        const unsigned step = (unsigned)pitch * sizeof(T);
        auto all = [&](unsigned thread, auto load) {
            const unsigned c = thread % kVecs * 8, at = thread / kVecs * step + c * (unsigned)sizeof(T);
#pragma unroll
            for (int k = 0; k < kPer; ++k)
                load(r[k], at + k * (THREADS / kVecs) * step, kUnits % THREADS == 0 || thread + k * THREADS < kUnits ? cols - (int)c : 0);
        };
        if (how == kAligned) {
            if (ANEW) asm volatile("" : "+v"(thread));
            all(thread, [&](Vec8<T>& v, unsigned at, int n) { load8(v, rsrc, at, n); });
            return;
        }
        // formed anew at every call: hoisted out of the chunk loop, these offsets and conditions would take a hundred registers
        asm volatile("" : "+v"(thread));
        if (how == kAnywhere && cols * (int)sizeof(T) >= 16) all(thread, [&](Vec8<T>& v, unsigned at, int n) { load8_anywhere(v, rsrc, at, n); });
        else all(thread, [&](Vec8<T>& v, unsigned at, int n) { load8_singly(v, rsrc, at, n); });
    }
    // whether this thread holds an infinity or a NaN: 0 times the sum of its values is not 0 then
    __device__ __forceinline__ bool odd() const {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) times_zero(r[k], v);
        return v != v;
    }
    // infinities and NaN become zeros; the first token of each value that had one goes to `token` (LDS)
    __device__ __forceinline__ void clear_odd(unsigned thread, int* token) {
        asm volatile("" : "+v"(thread));
#pragma unroll
        for (int k = 0; k < kPer; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = value(r[k], j);
                if (v - v == 0.f) continue;
                atomicMin(token + thread % kVecs * 8 + j, (int)(thread / kVecs + k * (THREADS / kVecs)));
                clear(r[k], j);
            }
    }
    template <Kind KIND>
    __device__ __forceinline__ void put(unsigned thread, Tile<T, kQ, COLS, KIND>& tile) const {
        const typename Tile<T, kQ, COLS, KIND>::Place place(thread / kVecs, thread % kVecs * 8);
        static_assert(THREADS / kVecs % 8 == 0, "a thread's rows are a multiple of 8 apart");
#pragma unroll
        for (int k = 0; k < kPer; ++k)
            if (kUnits % THREADS == 0 || thread + k * THREADS < kUnits) tile.put8(place, k * (THREADS / kVecs), r[k]);
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

// a lane's value in all lanes
__device__ __forceinline__ float lane_value(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }

__device__ __forceinline__ double lane_value(double v, int lane) {
    const long long bits = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_readlane((int)bits, lane), hi = __builtin_amdgcn_readlane((int)(bits >> 32), lane);
    return __builtin_bit_cast(double, (long long)(unsigned)lo | (long long)hi << 32);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
    const long long bits = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)bits, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(bits >> 32), CTRL, ROWS, 0xf, false);
    return v + __builtin_bit_cast(double, (long long)(unsigned)lo | (long long)hi << 32);
}
// sums over the lanes of this lane's row of 16: up to and including it, or from it on
__device__ __forceinline__ double row_sum_to(double v) {
    v = dpp_add<0x111, 0xf>(v);  // row_shr:1
    v = dpp_add<0x112, 0xf>(v);  // row_shr:2
    v = dpp_add<0x114, 0xf>(v);  // row_shr:4
    return dpp_add<0x118, 0xf>(v);  // row_shr:8
}
__device__ __forceinline__ double row_sum_from(double v) {
    v = dpp_add<0x101, 0xf>(v);  // row_shl:1
    v = dpp_add<0x102, 0xf>(v);  // row_shl:2
    v = dpp_add<0x104, 0xf>(v);  // row_shl:4
    return dpp_add<0x108, 0xf>(v);  // row_shl:8
}
// Sums over the tokens up to and including this lane's, in fp64: the differences s[t] - s[j] are what counts, and behind a strong decay both are large.
// Shifts inside the rows of 16 lanes, then the rows' last lanes handed on; lanes a step does not reach add 0.
__device__ __forceinline__ double running_sum(double v) {
    v = row_sum_to(v);
    v = dpp_add<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    return dpp_add<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
}
// Sums over the tokens from this lane's on, and those in front of it: of their own, not as what a sum over all leaves, which loses values 2^53 below the others
__device__ __forceinline__ double running_sum_from(double v) {
    v = row_sum_from(v);
    const int row = (threadIdx.x & 63) >> 4;
    const double t3 = lane_value(v, 48), t2 = lane_value(v, 32) + t3, t1 = lane_value(v, 16) + t2;
    return v + (row == 0 ? t1 : row == 1 ? t2 : row == 2 ? t3 : 0.0);
}
__device__ __forceinline__ double running_sum_before(double v) {
    v = running_sum(v);
    const long long bits = __builtin_bit_cast(long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)bits, 0x138, 0xf, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(bits >> 32), 0x138, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (long long)(unsigned)lo | (long long)hi << 32);  // wave_shr:1
}
// One wave, one token per lane: log2 decay (as two floats whose sum is the fp64 value to 48 bits).  A single token's is held at -4096: states are 0 behind it all the
// same (fp32 ends at -149), and the sums stay far from where fp32 ends, which rates of -1e38 would pass, and small enough that the decays behind it keep their bits.
__device__ __forceinline__ void chunk_decay(float step, float A, float& hi, float& lo) {
    const double v = (double)step * (double)A * 1.4426950408889634074, s = running_sum(v < -4096.0 ? -4096.0 : v);  // (a NaN goes through)
    hi = (float)s;
    lo = (float)(s - (double)hi);
}
// What the products of a chunk take from its decays, per token: s as two floats, d, e^{s[t]}, e^{s[63]-s[t]}
struct Decays {
    float hi[kQ], lo[kQ], step[kQ], from[kQ], to[kQ];
};

__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// by one wave for one chunk; `raw`: this lane's dt (with bias), `alive`: whether its token is within the row
struct Decay {
    float step, hi, lo;  // of this lane's token
    bool grows;          // whether any token of the chunk makes states larger
};
__device__ __forceinline__ Decay put_decays(Decays& o, float raw, bool alive, bool plus, float A) {
    const int lane = threadIdx.x & 63;
    Decay e;
    e.step = !alive ? 0.f : plus ? softplus(raw) : raw;
    e.grows = __ballot(e.step * A > 0.f) != 0;
    chunk_decay(e.step, A, e.hi, e.lo);
    const float eh = lane_value(e.hi, 63), el = lane_value(e.lo, 63);
    o.hi[lane] = e.hi, o.lo[lane] = e.lo, o.step[lane] = e.step, o.to[lane] = exp2_fast((eh - e.hi) + (el - e.lo));
    o.from[lane] = exp2_fast(e.hi) * fmaf(e.lo, 0.693147181f, 1.f);  // every token behind this one has the error of this
    return e;
}

// e^{s[t]-s[j]} of tokens in different tiles of 16 as a product of two factors with a decay s[r] between them: near[t] = e^{s[t]-s[r]} and
// to(tile of t)[j] = e^{s[r]-s[j]} weight[j], j in front of t's tile.  Where states only decay, r is the last token in front of t's tile, and both are at most 1.  Where
// they grow too, a factor could pass fp32's range though the product does not (0 times infinity): s[r] is halfway between the tile's largest s[t] and the smallest
// s[j] in front of it then, so that a factor is infinite only if the largest decay between the two sides passes e^176, and products of e^-43 and more keep both.
struct Factors {
    float near[kQ], far[16 + 32 + 48];  // far of the tiles 1, 2, 3 one behind the other
    __device__ __forceinline__ const float* to(int tile) const { return far + (tile == 1 ? 0 : tile == 2 ? 16 : 48); }
};
// the value of the lane BY places on, around this lane's row of 16
template <int BY> __device__ __forceinline__ float turned(float v) {
    const int bits = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(bits, bits, 0x120 + BY, 0xf, 0xf, false));  // row_ror
}
__device__ __forceinline__ void put_factors(Factors& o, const Decay& e, float weight) {
    const int lane = threadIdx.x & 63;
    float rh[3], rl[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) rh[k] = lane_value(e.hi, 16 * k + 15), rl[k] = lane_value(e.lo, 16 * k + 15);
    if (e.grows) {
        float top = e.hi, low = e.hi;
        top = fmaxf(top, turned<8>(top)), low = fminf(low, turned<8>(low));
        top = fmaxf(top, turned<4>(top)), low = fminf(low, turned<4>(low));
        top = fmaxf(top, turned<2>(top)), low = fminf(low, turned<2>(low));
        top = fmaxf(top, turned<1>(top)), low = fminf(low, turned<1>(low));
        float least = lane_value(low, 0);
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            rh[k] = 0.5f * (lane_value(top, 16 * (k + 1)) + least), rl[k] = 0.f;
            least = fminf(least, lane_value(low, 16 * (k + 1)));
        }
    }
    float nh = 0.f, nl = 0.f;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        if (lane <= 16 * k + 15) o.far[(k == 0 ? 0 : k == 1 ? 16 : 48) + lane] = exp2_fast((rh[k] - e.hi) + (rl[k] - e.lo)) * weight;
        if (lane >> 4 == k + 1) nh = rh[k], nl = rl[k];
    }
    o.near[lane] = exp2_fast((e.hi - nh) + (e.lo - nl));
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

// B H < 2^22: no launch, the step's with four workgroups per head included, reaches 2^32 threads
inline bool scan_sizes(int B, int L, int H, int P, int G, int N) {
    return B > 0 && L > 0 && L <= (1 << 30) && H > 0 && P > 0 && P <= 128 && G > 0 && H % G == 0 && N > 0 && N <= 128 && (long long)B * H < (1 << 22);
}

// 64 tokens must lie within 2^31 bytes of each other: buffer offsets
inline bool scan_pitch(long long tok) { return tok >= 0 && tok < (1ll << 23); }

void scan_cut(ScanArgs& a, int directions);
int scan_starts(const ScanArgs& a0, const ScanArgs& a1, const float* state1, float* ws, int both, int type, hipStream_t st);
int scan_walks(const ScanArgs& a0, const WalkOut& o0, const ScanArgs& a1, const WalkOut& o1, int both, int type, hipStream_t st);

inline ScanArgs scan_args(const void* x, long long x_row, long long x_tok, const Steps& dt, const float* A, const void* B, long long b_row, long long b_tok,
                          const void* C, long long c_row, long long c_tok, const float* D, const float* state, const int* lengths, int rows, int L, int H, int P,
                          int G, int N, int type, int directions) {
    ScanArgs a{x, B, C, x_row, x_tok, b_row, b_tok, c_row, c_tok, dt, A, D, state, lengths, rows, L, H, P, G, N, 1, 0, 0, 0, 0, 0, 0, 0, 0};
    const int v = type == 0 ? 4 : 8;  // values in 16 bytes
    auto how = [&](const void* p, int width, long long row, long long tok) {
        return width % v == 0 && row % v == 0 && tok % v == 0 && on16(p) ? kAligned : width >= v ? kAnywhere : kShort;
    };
    a.how_x = how(x, P, x_row, x_tok), a.how_b = how(B, N, b_row, b_tok), a.how_c = how(C, N, c_row, c_tok);
    scan_cut(a, directions);
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
