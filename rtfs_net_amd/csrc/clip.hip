// Global norm of many gradient tensors and their clipping to it (torch.nn.utils.clip_grad_norm_'s arithmetic; Lightning's gradient_clip_val: 5.0 in
// config yaml:117-120), for fp32, bf16 and fp16 tensors in any mix:
//   norm = (sum over all tensors of g^2)^(1/2)  or  max |g|,   g *= min(1, max_norm / (norm + 1e-6)).
// Bound: HBM for large lists (every gradient is read for the norm, read again and written), launches for small ones - RTFS-Net's 403 tensors are
// 740 k numbers.  The tensor list therefore travels in the kernel arguments (240 entries of 16 bytes per launch, below the 4 KB of an argument block):
// no table in device memory, no copy to it, and a captured graph holds all it needs.
// Squares are summed in fp64 from the first add on: the sum can neither overflow nor depend on the order beyond fp64's rounding, and a workgroup leaves
// ONE partial at a fixed place (no atomics), so the norm has the same bits on every run.  The scaling kernel sums the partials again in every workgroup (16 KB out
// of L2, ~1 us) instead of waiting for one more launch; lists of some 2000 tensors and more, whose launches leave more partials than that, take the launch.
// 300 M bf16 values in 291 tensors (1.8 GB read and written): 405 us, 4.4 TB/s; in 5000 tensors 651 us on the device, 2.1 ms on the
// host.  RTFS-Net's 403 tensors: 25 us on the device, 175 us on the host that lists them.
#include <algorithm>
#include <new>

#include "common.h"

namespace rtfs {

constexpr int kClipEntries = 240;       // tensors per launch
constexpr int kClipParts = 2048;        // workgroups of the whole list (8 per CU), and the most of one launch
constexpr int kClipLeast = 512;         // workgroups of a norm launch that has as many units, however long the list
constexpr int kClipFold = 4096;         // more partials than these are summed once, not by every workgroup
constexpr unsigned kClipUnit = 4096;    // elements a workgroup takes at a time
constexpr long long kClipLong = 1 << 30;  // a longer tensor is listed in pieces: element counts stay below 2^31

struct ClipList {
    unsigned long long at[kClipEntries];  // address of a piece's first element | type << 60 (addresses have 48 bits)
    unsigned n[kClipEntries];             // its elements
    unsigned end[kClipEntries];           // units up to and including it
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bhalf8 __attribute__((ext_vector_type(8)));
typedef float single4 __attribute__((ext_vector_type(4)));

template <typename T> struct ClipVec;
template <> struct ClipVec<float> { typedef single4 type; };
template <> struct ClipVec<__bf16> { typedef bhalf8 type; };
template <> struct ClipVec<_Float16> { typedef half8 type; };

// One unit of one piece.  Units are laid from the 16-byte line below the first element, so that whole vectors are aligned whatever the tensor's own
// alignment is (a view into a flat gradient buffer may start at any element); the vectors at the two ends are taken element by element.
template <typename T, bool SCALE, bool MAX>
__device__ __forceinline__ void clip_unit(T* g, unsigned n, unsigned unit, float coef, double& acc) {
    typedef typename ClipVec<T>::type Vec;
    constexpr int V = 16 / sizeof(T);
    const int before = (int)((reinterpret_cast<unsigned long long>(g) & 15) / sizeof(T));
    const long long first = (long long)unit * kClipUnit - before + (int)threadIdx.x * V;
    Vec v[kClipUnit / (256 * V)];
#pragma unroll
    for (int k = 0; k < (int)kClipUnit / (256 * V); ++k) {
        const long long i = first + (long long)k * 256 * V;
        if (i >= 0 && i + V <= n) {
            v[k] = *reinterpret_cast<const Vec*>(g + i);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[k][e] = i + e >= 0 && i + e < n ? g[i + e] : (T)0.f;
        }
    }
#pragma unroll
    for (int k = 0; k < (int)kClipUnit / (256 * V); ++k) {
        const long long i = first + (long long)k * 256 * V;
        if (SCALE) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[k][e] = (T)((float)v[k][e] * coef);
            if (i >= 0 && i + V <= n) {
                *reinterpret_cast<Vec*>(g + i) = v[k];
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (i + e >= 0 && i + e < n) g[i + e] = v[k][e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const double x = (double)(float)v[k][e];
                if (MAX) {
                    const double a = fabs(x);
                    acc = a > acc || a != a ? a : acc;  // a NaN stays (nothing compares above it)
                } else {
                    acc = fma(x, x, acc);
                }
            }
        }
    }
}

__device__ __forceinline__ double clip_join(double a, double b, bool max) {
    if (!max) return a + b;
    return b > a || b != b ? b : a;
}
// all 256 threads get the workgroup's total, in a fixed order
__device__ __forceinline__ double clip_reduce(double v, bool max, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = clip_join(v, __shfl_xor(v, o, 64), max);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return clip_join(clip_join(red[0], red[1], max), clip_join(red[2], red[3], max), max);
}

template <bool SCALE, bool MAX>
__global__ __launch_bounds__(256) void clip_kernel(ClipList list, int entries, double* __restrict__ parts, int n_parts, float max_norm, float* __restrict__ norm) {
    __shared__ double red[4];
    float coef = 1.f;
    if (SCALE) {
        double s = 0.0;
        for (int i = threadIdx.x; i < n_parts; i += 256) s = clip_join(s, parts[i], MAX);
        s = clip_reduce(s, MAX, red);
        const float total = (float)(MAX ? s : sqrt(s));
        if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
        coef = max_norm / (total + 1e-6f);
        coef = coef > 1.f ? 1.f : coef;  // a NaN goes through to every gradient
    }
    const unsigned units = list.end[entries - 1];
    const unsigned u0 = (unsigned)((unsigned long long)units * blockIdx.x / gridDim.x), u1 = (unsigned)((unsigned long long)units * (blockIdx.x + 1) / gridDim.x);
    int lo = 0, hi = entries - 1;  // the piece that holds unit u0
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list.end[mid] > u0) hi = mid;
        else lo = mid + 1;
    }
    double acc = 0.0;
    for (unsigned u = u0; u < u1; ++u) {
        while (list.end[lo] <= u) ++lo;
        const unsigned unit = u - (lo ? list.end[lo - 1] : 0u);
        const unsigned long long at = list.at[lo] & 0x0fffffffffffffffull;
        const int type = (int)(list.at[lo] >> 60);
        if (type == 0) clip_unit<float, SCALE, MAX>(reinterpret_cast<float*>(at), list.n[lo], unit, coef, acc);
        else if (type == 1) clip_unit<__bf16, SCALE, MAX>(reinterpret_cast<__bf16*>(at), list.n[lo], unit, coef, acc);
        else clip_unit<_Float16, SCALE, MAX>(reinterpret_cast<_Float16*>(at), list.n[lo], unit, coef, acc);
    }
    if (!SCALE) {
        acc = clip_reduce(acc, MAX, red);
        if (threadIdx.x == 0) parts[blockIdx.x] = acc;
    }
}

// the partials of a long list as one, in a fixed order
template <bool MAX>
__global__ __launch_bounds__(256) void clip_fold_kernel(const double* __restrict__ parts, int n_parts, double* __restrict__ total) {
    __shared__ double red[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < n_parts; i += 256) s = clip_join(s, parts[i], MAX);
    s = clip_reduce(s, MAX, red);
    if (threadIdx.x == 0) *total = s;
}

// Lists the tensors launch by launch; f(list, entries, units) for each full or last list.
template <typename F>
static void clip_lists(const long long* grads, const long long* sizes, const int* types, int n, ClipList& list, F f) {
    int k = 0;
    unsigned units = 0;
    for (int i = 0; i < n; ++i) {
        const int size = types[i] == 0 ? 4 : 2;
        for (long long from = 0; from < sizes[i]; from += kClipLong) {
            const long long left = sizes[i] - from, some = left < kClipLong ? left : kClipLong;
            const unsigned long long at = (unsigned long long)grads[i] + (unsigned long long)from * size;
            units += (unsigned)((some + (long long)((at & 15) / size) + kClipUnit - 1) / kClipUnit);
            list.at[k] = at | (unsigned long long)types[i] << 60;
            list.n[k] = (unsigned)some;
            list.end[k] = units;
            if (++k == kClipEntries) f(list, k, units), k = 0, units = 0;
        }
    }
    if (k) f(list, k, units);
}

// Whether two tensors have memory in common: their workgroups would scale it at once, in whatever order they run.  Lists in the order of their addresses, as
// views of one buffer come, are seen in one pass; others are sorted.  -> 0, 1, or -1 without memory to sort them in
static int clip_overlaps(const long long* grads, const long long* sizes, const int* types, int n) {
    struct Span {
        unsigned long long from, to;
        bool operator<(const Span& o) const { return from < o.from; }
    };
    auto span = [&](int i) { return Span{(unsigned long long)grads[i], (unsigned long long)grads[i] + (unsigned long long)sizes[i] * (types[i] == 0 ? 4 : 2)}; };
    unsigned long long end = 0;
    bool ordered = true;
    for (int i = 0; i < n && ordered; ++i) {
        if (!sizes[i]) continue;
        const Span s = span(i);
        ordered = s.from >= end, end = s.to;
    }
    if (ordered) return 0;
    Span* all = new (std::nothrow) Span[n];
    if (!all) return -1;
    int k = 0, found = 0;
    for (int i = 0; i < n; ++i)
        if (sizes[i]) all[k++] = span(i);
    std::sort(all, all + k);
    for (int i = 1; i < k; ++i) found |= all[i].from < all[i - 1].to;
    delete[] all;
    return found;
}

}  // namespace rtfs

using namespace rtfs;

extern "C" {

int rtfs_clip_grad_norm(const long long* grads, const long long* sizes, const int* types, int n, double max_norm, int norm_kind, double* parts, int n_parts,
                        float* norm, void* stream) {
    if (!grads || !sizes || !types || !parts || !norm || n <= 0 || (norm_kind != 0 && norm_kind != 2) || !(max_norm >= 0.0)) return RTFS_EINVAL;
    long long all = 0;
    for (int i = 0; i < n; ++i) {
        if (types[i] < 0 || types[i] > 2 || sizes[i] < 0 || (sizes[i] && (!grads[i] || grads[i] % (types[i] == 0 ? 4 : 2)))) return RTFS_EINVAL;
        all += sizes[i] / kClipUnit + 2;  // at least its units
    }
    if (clip_overlaps(grads, sizes, types, n)) return RTFS_EINVAL;
    ClipList list;
    // Workgroups of a norm launch: its share of kClipParts by its units, so that a list of few launches leaves few partials, but never so few that the card runs
    // empty: launches follow each other (300 M bf16 values in 5000 tensors: 1880 us on the device by shares alone, 651 so).  A scaling launch leaves none and takes
    // what it can use.
    auto groups = [&](unsigned units) {
        const long long share = (long long)kClipParts * units / all, most = share < kClipLeast ? kClipLeast : share;
        return (int)(most < units ? most : units);
    };
    int used = 0;
    clip_lists(grads, sizes, types, n, list, [&](const ClipList&, int, unsigned units) { used += groups(units); });
    const bool fold = used > kClipFold;
    if (used == 0 || used + fold > n_parts) return RTFS_EINVAL;
    int at = 0, failed = 0;
    clip_lists(grads, sizes, types, n, list, [&](const ClipList& l, int entries, unsigned units) {
        const dim3 grid(groups(units));
        if (norm_kind == 2)
            hipLaunchKernelGGL((clip_kernel<false, false>), grid, dim3(256), 0, (hipStream_t)stream, l, entries, parts + at, used, 0.f, (float*)nullptr);
        else
            hipLaunchKernelGGL((clip_kernel<false, true>), grid, dim3(256), 0, (hipStream_t)stream, l, entries, parts + at, used, 0.f, (float*)nullptr);
        at += (int)grid.x;
        failed |= hipGetLastError() != hipSuccess;
    });
    if (failed) return RTFS_ELAUNCH;
    if (fold) {
        if (norm_kind == 2) hipLaunchKernelGGL(clip_fold_kernel<false>, dim3(1), dim3(256), 0, (hipStream_t)stream, parts, used, parts + used);
        else hipLaunchKernelGGL(clip_fold_kernel<true>, dim3(1), dim3(256), 0, (hipStream_t)stream, parts, used, parts + used);
        RTFS_LAUNCH_CHECK();
        parts += used, used = 1;
    }
    float* out = norm;  // the first launch writes it
    clip_lists(grads, sizes, types, n, list, [&](const ClipList& l, int entries, unsigned units) {
        const dim3 grid(units < (unsigned)kClipParts ? units : (unsigned)kClipParts);
        if (norm_kind == 2)
            hipLaunchKernelGGL((clip_kernel<true, false>), grid, dim3(256), 0, (hipStream_t)stream, l, entries, parts, used, (float)max_norm, out);
        else
            hipLaunchKernelGGL((clip_kernel<true, true>), grid, dim3(256), 0, (hipStream_t)stream, l, entries, parts, used, (float)max_norm, out);
        out = nullptr;
        failed |= hipGetLastError() != hipSuccess;
    });
    return failed ? RTFS_ELAUNCH : RTFS_OK;
}

}  // extern "C"
