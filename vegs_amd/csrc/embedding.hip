// embedding.hip -- the row lookup and its gradients (include/vegs_embedding.h).
#include "../../include/vegs_embedding.h"
#include "vr_host.h"
#include "vr_types.h"

namespace vr {

struct LookupArgs {
    const void* table;
    const void* ids;
    const float* row_scale;
    long n, rows, width, table_stride;
    int ids_64;
    float scale;
};

// the row of entry i, or -1
__device__ __forceinline__ long row_of(const LookupArgs& a, long i)
{
    const long id = a.ids_64 ? (long)reinterpret_cast<const int64_t*>(a.ids)[i] : (long)reinterpret_cast<const int32_t*>(a.ids)[i];
    return id >= 0 && id < a.rows ? id : -1;
}

template <typename TT, typename TO>
__global__ void __launch_bounds__(256) k_lookup_fwd(LookupArgs a, TO* __restrict__ out)
{
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    if (e >= a.n * a.width) return;
    const long i = e / a.width, c = e - i * a.width;
    const long row = row_of(a, i);
    float x = 0.0f;
    if (row >= 0) {
        x = load_f32(reinterpret_cast<const TT*>(a.table) + row * a.table_stride + c);
        if (a.row_scale) x *= a.scale * a.row_scale[i];
        else x *= a.scale;
    }
    store_f32(out + e, x);
}

// sort keys: the row, or `rows` for "no row" (sorted behind every row); values: the entry
__global__ void __launch_bounds__(256) k_lookup_keys(LookupArgs a, uint32_t* __restrict__ key, uint32_t* __restrict__ val)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.n) return;
    const long row = row_of(a, i);
    key[i] = row >= 0 ? (uint32_t)row : (uint32_t)a.rows;
    val[i] = (uint32_t)i;
}

__device__ __forceinline__ long lower_bound(const uint32_t* key, long n, uint32_t k)
{
    long lo = 0, hi = n;
    while (lo < hi) {
        const long mid = (lo + hi) >> 1;
        if (key[mid] < k) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// one wave per row of the table: the row's entries one after the other, lanes across the columns
template <typename TT, typename TO>
__global__ void __launch_bounds__(64)
k_lookup_sum(LookupArgs a, const TO* __restrict__ grad, long grad_stride, const uint32_t* __restrict__ key,
             const uint32_t* __restrict__ val, TT* __restrict__ d_table)
{
    const long row = blockIdx.x;
    const long first = lower_bound(key, a.n, (uint32_t)row), last = lower_bound(key, a.n, (uint32_t)row + 1);
    for (long c = threadIdx.x; c < a.width; c += 64) {
        float acc = 0.0f;
        for (long j = first; j < last; ++j) {
            const long i = val[j];
            const float s = a.row_scale ? a.scale * a.row_scale[i] : a.scale;
            acc = fmaf(s, load_f32(grad + i * grad_stride + c), acc);
        }
        store_f32(d_table + row * a.width + c, acc);
    }
}

// one wave per entry
template <typename TT, typename TO>
__global__ void __launch_bounds__(64)
k_lookup_dscale(LookupArgs a, const TO* __restrict__ grad, long grad_stride, float* __restrict__ d_row_scale)
{
    const long i = blockIdx.x, row = row_of(a, i);
    float acc = 0.0f;
    if (row >= 0)
        for (long c = threadIdx.x; c < a.width; c += 64)
            acc = fmaf(load_f32(grad + i * grad_stride + c),
                       load_f32(reinterpret_cast<const TT*>(a.table) + row * a.table_stride + c), acc);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) acc += __shfl_xor(acc, d, 64);
    if (threadIdx.x == 0) d_row_scale[i] = a.scale * acc;
}

static int check_lookup(const VrLookup* l, LookupArgs& a)
{
    if (!l) { set_error("lookup: arguments are required"); return VR_ERR_INVALID_ARGUMENT; }
    if (l->n < 0 || l->n >= (1ll << 30) || l->rows < 0 || l->rows >= 0x7fffffffll || l->width < 1 || l->width > (1 << 24) ||
        l->table_stride < l->width || l->table_stride > (1ll << 40))
        { set_error("lookup: need 0 <= n < 2^30, 0 <= rows < 2^31 - 1, 1 <= width <= 2^24, table_stride >= width"); return VR_ERR_INVALID_ARGUMENT; }
    if (l->table_dtype < VR_F32 || l->table_dtype > VR_F16 || (l->out_dtype != l->table_dtype && l->out_dtype != VR_F32))
        { set_error("lookup: the output has the table's type or fp32"); return VR_ERR_INVALID_ARGUMENT; }
    const uintptr_t element = l->table_dtype == VR_F32 ? 4 : 2, id = l->ids_64 ? 8 : 4;
    if ((l->n > 0 && !l->ids) || (l->n > 0 && l->rows > 0 && !l->table) || ((uintptr_t)l->table & (element - 1)) ||
        ((uintptr_t)l->ids & (id - 1)) || ((uintptr_t)l->row_scale & 3))
        { set_error("lookup: table and ids are required, aligned to their elements"); return VR_ERR_INVALID_ARGUMENT; }
    a = LookupArgs{l->table, l->ids, l->row_scale, (long)l->n, (long)l->rows, (long)l->width, (long)l->table_stride,
                   l->ids_64 != 0, l->scale};
    return VR_OK;
}

static int key_bits(int64_t rows)            // of the keys 0 .. rows
{
    int b = 0;
    while (b < 32 && (rows >> b) != 0) ++b;
    return b;
}

// calls F::template run<table type, output type>(...)
template <typename F, typename... A>
static int by_type(const VrLookup* l, A... args)
{
    if (l->table_dtype == VR_F32) return F::template run<float, float>(args...);
    if (l->table_dtype == VR_BF16) return l->out_dtype == VR_F32 ? F::template run<bf16, float>(args...) : F::template run<bf16, bf16>(args...);
    return l->out_dtype == VR_F32 ? F::template run<__half, float>(args...) : F::template run<__half, __half>(args...);
}

struct Forward {
    template <typename TT, typename TO>
    static int run(const LookupArgs& a, void* out, hipStream_t s)
    {
        const long blocks = (a.n * a.width + 255) / 256;
        if (blocks > 0x7fffffffl) { set_error("lookup: n x width is too large"); return VR_ERR_INVALID_ARGUMENT; }
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_fwd<TT, TO>), dim3((unsigned)blocks), dim3(256), 0, s, a, (TO*)out);
        if (hipGetLastError() != hipSuccess) { set_error("lookup: kernel launch failed"); return VR_ERR_HIP; }
        return VR_OK;
    }
};

struct Backward {
    template <typename TT, typename TO>
    static int run(const LookupArgs& a, const void* grad, long grad_stride, const uint32_t* key, const uint32_t* val, void* d_table,
                   float* d_row_scale, hipStream_t s)
    {
        if (d_table && a.rows > 0)
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_sum<TT, TO>), dim3((unsigned)a.rows), dim3(64), 0, s, a, (const TO*)grad,
                               grad_stride, key, val, (TT*)d_table);
        if (d_row_scale && a.n > 0)
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_dscale<TT, TO>), dim3((unsigned)a.n), dim3(64), 0, s, a, (const TO*)grad,
                               grad_stride, d_row_scale);
        if (hipGetLastError() != hipSuccess) { set_error("lookup: kernel launch failed"); return VR_ERR_HIP; }
        return VR_OK;
    }
};

}  // namespace vr

using namespace vr;

extern "C" int vr_lookup_forward(const VrLookup* lookup, void* out, void* stream)
{
    LookupArgs a;
    if (int rc = check_lookup(lookup, a)) return rc;
    const uintptr_t element = lookup->out_dtype == VR_F32 ? 4 : 2;
    if (a.n > 0 && (!out || ((uintptr_t)out & (element - 1)))) { set_error("lookup: out is required, aligned to its elements"); return VR_ERR_INVALID_ARGUMENT; }
    if (a.n == 0) return VR_OK;
    return by_type<Forward>(lookup, a, out, (hipStream_t)stream);
}

extern "C" int64_t vr_lookup_scratch_bytes(int64_t n, int64_t rows, int64_t width)
{
    if (n < 0 || n >= (1ll << 30) || rows < 0 || rows >= 0x7fffffffll || width < 1 || width > (1 << 24)) return 0;
    return (int64_t)(4 * align_up((size_t)(n > 0 ? n : 1) * 4, 256) + sort_pairs_scratch_bytes((long)n));
}

extern "C" int vr_lookup_backward(const VrLookup* lookup, const void* grad, int64_t grad_stride, void* d_table, float* d_row_scale,
                                  void* scratch, int64_t scratch_bytes, void* stream)
{
    LookupArgs a;
    if (int rc = check_lookup(lookup, a)) return rc;
    const uintptr_t element = lookup->out_dtype == VR_F32 ? 4 : 2, t_element = lookup->table_dtype == VR_F32 ? 4 : 2;
    if ((a.n > 0 && !grad) || ((uintptr_t)grad & (element - 1)) || grad_stride < a.width || grad_stride > (1ll << 40) ||
        ((uintptr_t)d_table & (t_element - 1)) || ((uintptr_t)d_row_scale & 3))
        { set_error("lookup: grad is required, arrays aligned to their elements, grad_stride >= width"); return VR_ERR_INVALID_ARGUMENT; }
    if (d_table && (!scratch || ((uintptr_t)scratch & 255) || scratch_bytes < vr_lookup_scratch_bytes(a.n, a.rows, a.width)))
        { set_error("lookup: the table's gradient needs vr_lookup_scratch_bytes of scratch, 256-byte aligned"); return VR_ERR_INVALID_ARGUMENT; }
    if ((!d_table || a.rows == 0) && (!d_row_scale || a.n == 0)) return VR_OK;
    hipStream_t s = (hipStream_t)stream;
    const uint32_t *key = nullptr, *val = nullptr;
    if (d_table && a.n > 0) {
        const size_t arr = align_up((size_t)a.n * 4, 256);
        char* base = (char*)scratch;
        uint32_t *k0 = (uint32_t*)base, *v0 = (uint32_t*)(base + arr), *k1 = (uint32_t*)(base + 2 * arr), *v1 = (uint32_t*)(base + 3 * arr);
        hipLaunchKernelGGL(k_lookup_keys, dim3(cdiv(a.n, 256)), dim3(256), 0, s, a, k0, v0);
        VR_KERNEL_CHECK("lookup_keys", s, false);
        int where = 0;
        if (int rc = launch_sort_pairs(k0, v0, k1, v1, a.n, 0u, key_bits(a.rows), base + 4 * arr, s, false, &where)) return rc;
        key = where ? k1 : k0;
        val = where ? v1 : v0;
    }
    return by_type<Backward>(lookup, a, grad, (long)grad_stride, key, val, d_table, d_row_scale, s);
}
