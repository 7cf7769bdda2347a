// gradnorm.hip -- the global gradient norm over many tensors, and clipping (include/vegs_optim.h).
//
//   norm = sqrt(sum over all tensors of g^2)   or   max |g|;      g *= min(1, max_norm / (norm + 1e-6))
//
// Bound by HBM: the norm reads every gradient once, the scaling reads and writes it once more, and only when the factor is not
// one (118 M fp32 elements: 76 us, 6.2 TB/s, and 150 us, 6.3 TB/s).  The squares are taken and added in fp64: a product of two
// fp32 values is exact there and neither overflows nor vanishes, and the vector ALUs do 64-bit multiply-adds an order of
// magnitude faster than memory delivers operands.  No atomics: every workgroup writes one partial result, and they are added in
// one fixed order, so that the ranks of a job that hold the same gradients clip by the same bits.
#include "../../include/vegs_optim.h"
#include "vr_host.h"
#include "vr_sh_factors.h"
#include "vr_types.h"

#include <algorithm>
#include <new>

namespace vr {

constexpr int GN_MAX_T = 128;              // tensors per launch: the table is a kernel argument, 128 x 24 B of its 4 KB
// A thread has two 16-byte loads in flight, a workgroup's unit is 8 KB, and 1024 workgroups -- four for each of the 256 CUs -- go
// through the units in turns.  (118 M fp32 elements: 76 us; with 2048 workgroups 81 for two, four and eight loads alike.  18 M bf16
// elements, the largest magnitude: 11 us, 14 for four loads, 21 for eight, whose unpacked values wait on one another.)
constexpr int GN_LOADS = 2, GN_UNIT = GN_LOADS * 256 * 16, GN_GRID = 1024;

struct GradSeg {
    void* data;
    long n;
    int unit0;             // first unit of this tensor
    int dtype;
};
struct GradArgs {
    GradSeg seg[GN_MAX_T];
    int count, units;
};

// 16 bytes of values at an address of their own alignment (a gradient may be a view that starts anywhere)
template <typename T>
struct __attribute__((packed)) Quad { T v[16 / sizeof(T)]; };

// the norm's accumulator: a sum of squares in fp64, or the largest magnitude in fp32 (a NaN, once met, stays)
template <bool MAX> struct Acc { using type = double; };
template <> struct Acc<true> { using type = float; };

__device__ __forceinline__ double norm_add(double acc, float x) { return fma((double)x, (double)x, acc); }
__device__ __forceinline__ double norm_join(double a, double b) { return a + b; }
__device__ __forceinline__ float norm_join(float a, float b) { return (b > a || b != b) ? b : a; }
__device__ __forceinline__ float norm_add(float acc, float x) { return norm_join(acc, fabsf(x)); }
__device__ __forceinline__ float norm_value(double acc) { return (float)sqrt(acc); }
__device__ __forceinline__ float norm_value(float acc) { return acc; }

// over the workgroup's waves, in a fixed order; the result is thread 0's.  lds: one value per wave
template <typename T>
__device__ __forceinline__ T norm_block(T acc, T* lds)
{
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) acc = norm_join(acc, __shfl_xor(acc, d, 64));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < (int)(blockDim.x >> 6); ++w) acc = norm_join(acc, lds[w]);
    return acc;
}
// the workgroups' partial results, by one workgroup of 256 threads: always in this order
template <bool MAX>
__device__ __forceinline__ float norm_total(const double* __restrict__ partial, int n, typename Acc<MAX>::type* lds)
{
    typename Acc<MAX>::type acc = 0;
    for (int i = threadIdx.x; i < n; i += 256) acc = norm_join(acc, (typename Acc<MAX>::type)partial[i]);
    return norm_value(norm_block(acc, lds));
}

__device__ __forceinline__ GradSeg grad_seg(const GradArgs& a, int unit)
{
    int t = 0, hi = a.count - 1;          // the last tensor whose first unit is <= unit (scalar binary search)
    while (t < hi) {
        const int mid = (t + hi + 1) >> 1;
        if (unit >= a.seg[mid].unit0) t = mid; else hi = mid - 1;
    }
    return a.seg[t];
}

// A unit's values: the thread's loads at once where the unit is full, single values in a tensor's last unit.
// Two accumulators, for the 64-bit multiply-add's latency.
template <typename T, typename A>
__device__ __forceinline__ void norm_unit(const void* data, long base, long n, A& acc0, A& acc1)
{
    constexpr int V = 16 / sizeof(T), PER = 256 * V;
    const T* p = reinterpret_cast<const T*>(data) + base;
    const long left = n - base;
    if (left >= GN_LOADS * PER) {
        Quad<T> q[GN_LOADS];
#pragma unroll
        for (int j = 0; j < GN_LOADS; ++j) q[j] = *reinterpret_cast<const Quad<T>*>(p + j * PER + threadIdx.x * V);
#pragma unroll
        for (int j = 0; j < GN_LOADS; ++j)
#pragma unroll
            for (int v = 0; v < V; v += 2) {
                acc0 = norm_add(acc0, load_f32(q[j].v + v));
                acc1 = norm_add(acc1, load_f32(q[j].v + v + 1));
            }
    } else {
        for (long i = threadIdx.x; i < left; i += 256) acc0 = norm_add(acc0, load_f32(p + i));      // (less than a unit)
    }
}

template <bool MAX>
__global__ void __launch_bounds__(256) k_grad_norm(GradArgs a, double* __restrict__ partial)
{
    using A = typename Acc<MAX>::type;
    __shared__ A lds[4];
    A acc = 0, acc1 = 0;
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const GradSeg s = grad_seg(a, unit);
        const long at = (long)(unit - s.unit0) * GN_UNIT;
        if (s.dtype == VR_F32) norm_unit<float>(s.data, at / 4, s.n, acc, acc1);
        else if (s.dtype == VR_BF16) norm_unit<bf16>(s.data, at / 2, s.n, acc, acc1);
        else norm_unit<__half>(s.data, at / 2, s.n, acc, acc1);
    }
    acc = norm_block(norm_join(acc, acc1), lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// (2 M Gaussians, degree 3: 22 us for one view, 41 for four, where the bytes take 9 and 23 at a copy's rate: one Gaussian's loads in
// flight a thread, and the 48 squares one after the other; the dense gradient would be 384 MB to write and read.)
// One Gaussian per thread: its dense SH row is rebuilt in registers, from the same function the optimizer's kernel
// steps with, and only its squares leave.
template <bool MAX>
__global__ void __launch_bounds__(256) k_sh_grad_norm(ShFactorArgs a, double* __restrict__ partial)
{
    using A = typename Acc<MAX>::type;
    __shared__ A lds[4];
    A acc = 0;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < a.P; i += gridDim.x * 256) {
        float g[SHF_ROW_MAX];
#pragma unroll
        for (int q = 0; q < SHF_ROW_MAX; ++q) g[q] = 0.0f;
        sh_row_from_factors(a, (int)i, g);
#pragma unroll
        for (int q = 0; q < SHF_ROW_MAX; ++q) acc = norm_add(acc, a.scale * g[q]);
    }
    acc = norm_block(acc, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

template <bool MAX>
__global__ void __launch_bounds__(256) k_grad_norm_finish(const double* __restrict__ partial, int n, float* __restrict__ norm)
{
    __shared__ typename Acc<MAX>::type lds[4];
    const float x = norm_total<MAX>(partial, n, lds);
    if (threadIdx.x == 0) norm[0] = x;
}

template <typename T>
__device__ __forceinline__ void scale_unit(void* data, long base, long n, float c)
{
    constexpr int V = 16 / sizeof(T), PER = 256 * V;
    T* p = reinterpret_cast<T*>(data) + base;
    const long left = n - base;
    if (left >= GN_LOADS * PER) {
        Quad<T> q[GN_LOADS];
#pragma unroll
        for (int j = 0; j < GN_LOADS; ++j) q[j] = *reinterpret_cast<const Quad<T>*>(p + j * PER + threadIdx.x * V);
#pragma unroll
        for (int j = 0; j < GN_LOADS; ++j) {
#pragma unroll
            for (int v = 0; v < V; ++v) store_f32(q[j].v + v, c * load_f32(q[j].v + v));
            *reinterpret_cast<Quad<T>*>(p + j * PER + threadIdx.x * V) = q[j];
        }
    } else {
        for (long i = threadIdx.x; i < left; i += 256) store_f32(p + i, c * load_f32(p + i));
    }
}

// The norm comes from memory, or (KIND 1: sum of squares, 2: largest magnitude) from k_grad_norm's partial results, which every workgroup
// adds up for itself -- 8 KB a launch from the L2 each, and a launch less between the two passes.
template <int KIND>
__global__ void __launch_bounds__(256) k_clip_grads(GradArgs a, float* __restrict__ norm, float max_norm,
                                                    const double* __restrict__ partial, int n_partial)
{
    float c;
    if (KIND) {
        __shared__ typename Acc<KIND == 2>::type lds[4];
        __shared__ float total;
        const float x = norm_total<KIND == 2>(partial, n_partial, lds);
        if (threadIdx.x == 0) {
            total = x;
            if (blockIdx.x == 0) norm[0] = x;
        }
        __syncthreads();
        c = clip_factor(total, max_norm);
    } else {
        c = clip_factor(*norm, max_norm);
    }
    if (c == 1.0f) return;
    for (int unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
        const GradSeg s = grad_seg(a, unit);
        const long at = (long)(unit - s.unit0) * GN_UNIT;
        if (s.dtype == VR_F32) scale_unit<float>(s.data, at / 4, s.n, c);
        else if (s.dtype == VR_BF16) scale_unit<bf16>(s.data, at / 2, s.n, c);
        else scale_unit<__half>(s.data, at / 2, s.n, c);
    }
}

// A handful of small tensors -- the pose corrections of a frame -- by one workgroup: a wave per tensor, the norm, and (CLIP)
// the scaling, in one launch instead of three.
constexpr int GN_SMALL = 2048;             // values of one tensor, at most: 32 a lane
constexpr int GN_SMALL_ALL = 16384;        // of all of them
template <bool MAX, bool CLIP>
__global__ void __launch_bounds__(1024) k_grad_norm_small(GradArgs a, float max_norm, float* __restrict__ norm)
{
    using A = typename Acc<MAX>::type;
    __shared__ A lds[16];
    __shared__ float factor;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    A acc = 0;
    for (int t = w; t < a.count; t += 16) {
        const GradSeg s = a.seg[t];
        for (int i = lane; i < (int)s.n; i += 64)
            acc = norm_add(acc, s.dtype == VR_F32 ? load_f32(reinterpret_cast<const float*>(s.data) + i)
                                     : s.dtype == VR_BF16 ? load_f32(reinterpret_cast<const bf16*>(s.data) + i)
                                                          : load_f32(reinterpret_cast<const __half*>(s.data) + i));
    }
    acc = norm_block(acc, lds);
    if (threadIdx.x == 0) {
        const float x = norm_value(acc);
        norm[0] = x;
        factor = CLIP ? clip_factor(x, max_norm) : 1.0f;
    }
    if (!CLIP) return;
    __syncthreads();
    const float c = factor;
    if (c == 1.0f) return;
    for (int t = w; t < a.count; t += 16) {
        const GradSeg s = a.seg[t];
        for (int i = lane; i < (int)s.n; i += 64) {
            if (s.dtype == VR_F32) { float* p = reinterpret_cast<float*>(s.data) + i; store_f32(p, c * load_f32(p)); }
            else if (s.dtype == VR_BF16) { bf16* p = reinterpret_cast<bf16*>(s.data) + i; store_f32(p, c * load_f32(p)); }
            else { __half* p = reinterpret_cast<__half*>(s.data) + i; store_f32(p, c * load_f32(p)); }
        }
    }
}

static bool small_grads(const VrGradTensor* t, int32_t count)
{
    int64_t all = 0, used = 0;
    for (int i = 0; i < count; ++i) {
        if (t[i].n > GN_SMALL) return false;
        all += t[i].n;
        used += t[i].n > 0;
    }
    return used <= GN_MAX_T && all <= GN_SMALL_ALL;
}

static int check_grads(const VrGradTensor* t, int32_t count)
{
    if (count < 0 || (count > 0 && !t)) { set_error("grad norm: bad tensor list"); return VR_ERR_INVALID_ARGUMENT; }
    for (int i = 0; i < count; ++i) {
        if (t[i].dtype < VR_F32 || t[i].dtype > VR_F16) { set_error("grad norm: tensor %d has an unknown type", i); return VR_ERR_INVALID_ARGUMENT; }
        const uintptr_t element = t[i].dtype == VR_F32 ? 4 : 2;
        // (one tensor's units are counted in 31 bits: 2^40 values are 2^29 of them)
        if (t[i].n < 0 || (t[i].n > 0 && (!t[i].data || ((uintptr_t)t[i].data & (element - 1)))) || t[i].n > (1ll << 40))
            { set_error("grad norm: tensor %d with NULL or misaligned data or a bad size", i); return VR_ERR_INVALID_ARGUMENT; }
    }
    return VR_OK;
}

// Whether no two of the tensors share memory: workgroups scale units of different tensors side by side, and an element that two
// of them hold would be read, multiplied and written by both.
static int check_apart(const VrGradTensor* t, int32_t count)
{
    struct Range { uintptr_t begin, end; int at; };
    Range few[GN_MAX_T];
    Range* r = count <= GN_MAX_T ? few : new (std::nothrow) Range[count];
    if (!r) { set_error("clip: no memory for a list of %d tensors", count); return VR_ERR_ALLOC; }
    int n = 0;
    for (int i = 0; i < count; ++i)
        if (t[i].n > 0) {
            const uintptr_t at = (uintptr_t)t[i].data;
            r[n++] = Range{at, at + (uintptr_t)t[i].n * (t[i].dtype == VR_F32 ? 4 : 2), i};
        }
    std::sort(r, r + n, [](const Range& a, const Range& b) { return a.begin < b.begin; });
    int rc = VR_OK;
    for (int i = 1; i < n && rc == VR_OK; ++i)
        if (r[i].begin < r[i - 1].end) {
            set_error("clip: tensors %d and %d share memory", std::min(r[i - 1].at, r[i].at), std::max(r[i - 1].at, r[i].at));
            rc = VR_ERR_INVALID_ARGUMENT;
        }
    if (r != few) delete[] r;
    return rc;
}

// the next launch's table: up to GN_MAX_T non-empty tensors from `first` on; returns the first one not consumed
static int fill_grads(const VrGradTensor* t, int first, int count, GradArgs& a)
{
    int next = first;
    a.count = a.units = 0;
    for (; next < count && a.count < GN_MAX_T; ++next) {
        if (t[next].n == 0) continue;
        const long units = (t[next].n * (t[next].dtype == VR_F32 ? 4 : 2) + GN_UNIT - 1) / GN_UNIT;
        if (a.units + units > 0x3fffffff) break;
        a.seg[a.count++] = GradSeg{t[next].data, (long)t[next].n, a.units, (int)t[next].dtype};
        a.units += (int)units;
    }
    for (int i = a.count; i < GN_MAX_T; ++i) a.seg[i] = GradSeg{nullptr, 0, 0x7fffffff, 0};
    return next;
}

template <int KIND>
static void launch_clip(const GradArgs& a, float* norm, float max_norm, const double* partial, int n, hipStream_t s)
{
    hipLaunchKernelGGL(k_clip_grads<KIND>, dim3(a.units < GN_GRID ? a.units : GN_GRID), dim3(256), 0, s, a, norm, max_norm, partial, n);
}

// clip: scale as well
template <bool MAX>
static int grad_norm(const VrGradTensor* tensors, int32_t count, const VrShGradFactors* factors, int32_t n_factors,
                     float* norm, double* partial, hipStream_t s, bool clip = false, float max_norm = 0.0f)
{
    int n = 0;
    if (n_factors == 0 && small_grads(tensors, count)) {
        GradArgs a;
        fill_grads(tensors, 0, count, a);
        if (clip) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_grad_norm_small<MAX, true>), dim3(1), dim3(1024), 0, s, a, max_norm, norm);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_grad_norm_small<MAX, false>), dim3(1), dim3(1024), 0, s, a, max_norm, norm);
        if (hipGetLastError() != hipSuccess) { set_error("grad norm: kernel launch failed"); return VR_ERR_HIP; }
        return VR_OK;
    }
    for (int first = 0; first < count;) {
        GradArgs a;
        first = fill_grads(tensors, first, count, a);
        if (a.units == 0) continue;
        const int grid = a.units < GN_GRID ? a.units : GN_GRID;
        hipLaunchKernelGGL(k_grad_norm<MAX>, dim3(grid), dim3(256), 0, s, a, partial + n);
        n += grid;
    }
    for (int i = 0; i < n_factors; ++i) {
        const VrShGradFactors& f = factors[i];
        ShFactorArgs a;
        if (int rc = sh_factor_args(a, f.means3D, f.P, f.campos, f.factors, f.n_views, f.factor_view_stride, f.sh_degree,
                                    (f.sh_degree + 1) * (f.sh_degree + 1), f.scale)) return rc;
        if (f.P == 0) continue;
        const int grid = cdiv(f.P, 256) < GN_GRID ? cdiv(f.P, 256) : GN_GRID;
        hipLaunchKernelGGL(k_sh_grad_norm<MAX>, dim3(grid), dim3(256), 0, s, a, partial + n);
        n += grid;
    }
    if (clip && n > 0) {
        for (int first = 0; first < count;) {
            GradArgs a;
            first = fill_grads(tensors, first, count, a);
            if (a.units > 0) launch_clip<MAX ? 2 : 1>(a, norm, max_norm, partial, n, s);
        }
    } else {
        hipLaunchKernelGGL(k_grad_norm_finish<MAX>, dim3(1), dim3(256), 0, s, (const double*)partial, n, norm);
    }
    if (hipGetLastError() != hipSuccess) { set_error("grad norm: kernel launch failed"); return VR_ERR_HIP; }
    return VR_OK;
}

static int clip_grads(const VrGradTensor* tensors, int32_t count, const float* norm, float max_norm, hipStream_t s)
{
    for (int first = 0; first < count;) {
        GradArgs a;
        first = fill_grads(tensors, first, count, a);
        if (a.units > 0) launch_clip<0>(a, const_cast<float*>(norm), max_norm, nullptr, 0, s);
    }
    if (hipGetLastError() != hipSuccess) { set_error("clip: kernel launch failed"); return VR_ERR_HIP; }
    return VR_OK;
}

}  // namespace vr

using namespace vr;

// (a launch takes fewer than GN_MAX_T tensors only when its units run out, at 8 TB of gradients)
extern "C" int64_t vr_grad_norm_scratch_bytes(int32_t count, int32_t n_factors)
{
    const int64_t launches = (count > 0 ? (count + GN_MAX_T - 1) / GN_MAX_T : 0) + (n_factors > 0 ? n_factors : 0);
    return (launches > 0 ? launches : 1) * GN_GRID * (int64_t)sizeof(double);
}

static int check_norm(const VrGradTensor* tensors, int32_t count, const VrShGradFactors* factors, int32_t n_factors,
                      int32_t norm_type, const float* norm, const void* scratch)
{
    if (int rc = check_grads(tensors, count)) return rc;
    if (n_factors < 0 || (n_factors > 0 && !factors) || !norm || !scratch || ((uintptr_t)scratch & 7) || (norm_type != 2 && norm_type != 0))
        { set_error("grad norm: needs norm, 8-byte aligned scratch and norm_type 2 or 0 (largest magnitude)"); return VR_ERR_INVALID_ARGUMENT; }
    for (int i = 0; i < n_factors; ++i) {                  // everything is checked before anything is launched
        const VrShGradFactors& f = factors[i];
        ShFactorArgs a;
        if (int rc = sh_factor_args(a, f.means3D, f.P, f.campos, f.factors, f.n_views, f.factor_view_stride, f.sh_degree,
                                    (f.sh_degree + 1) * (f.sh_degree + 1), f.scale)) return rc;
    }
    return VR_OK;
}

extern "C" int vr_grad_norm(const VrGradTensor* tensors, int32_t count, const VrShGradFactors* factors, int32_t n_factors,
                            int32_t norm_type, float* norm, void* scratch, void* stream)
{
    if (int rc = check_norm(tensors, count, factors, n_factors, norm_type, norm, scratch)) return rc;
    return norm_type == 2 ? grad_norm<false>(tensors, count, factors, n_factors, norm, (double*)scratch, (hipStream_t)stream)
                          : grad_norm<true>(tensors, count, factors, n_factors, norm, (double*)scratch, (hipStream_t)stream);
}

extern "C" int vr_clip_grads(const VrGradTensor* tensors, int32_t count, const float* norm, float max_norm, void* stream)
{
    if (int rc = check_grads(tensors, count)) return rc;
    if (!norm || !(max_norm >= 0.0f)) { set_error("clip: needs a norm and max_norm >= 0"); return VR_ERR_INVALID_ARGUMENT; }
    if (int rc = check_apart(tensors, count)) return rc;
    return clip_grads(tensors, count, norm, max_norm, (hipStream_t)stream);
}

extern "C" int vr_clip_grad_norm(const VrGradTensor* tensors, int32_t count, int32_t norm_type, float max_norm, float* norm,
                                 void* scratch, void* stream)
{
    if (!(max_norm >= 0.0f)) { set_error("clip: max_norm must not be negative or NaN"); return VR_ERR_INVALID_ARGUMENT; }
    if (int rc = check_norm(tensors, count, nullptr, 0, norm_type, norm, scratch)) return rc;
    if (int rc = check_apart(tensors, count)) return rc;
    return norm_type == 2 ? grad_norm<false>(tensors, count, nullptr, 0, norm, (double*)scratch, (hipStream_t)stream, true, max_norm)
                          : grad_norm<true>(tensors, count, nullptr, 0, norm, (double*)scratch, (hipStream_t)stream, true, max_norm);
}
