// embedding.hip -- the row lookup and its gradients (include/vegs_embedding.h).
#include "../../include/vegs_embedding.h"
#include "vr_host.h"
#include "vr_types.h"

#include <type_traits>

namespace vr {

struct LookupArgs {
    const void* table;
    const void* ids;
    const float* row_scale;
    long n, rows, width, table_stride;
    int ids_64;
    float scale;
};

// V values that lie next to each other, at any address their type may have: one load or store of up to 16 bytes
template <typename T, int V>
struct __attribute__((packed)) Pack { T v[V]; };

// 16 bytes at an address of 2 or 4 bytes' alignment, past the caches' normal order of replacement
typedef uint32_t quad_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t quad_2 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_once(const T* p)
{
    if (sizeof(Pack<T, V>) != 16) return *reinterpret_cast<const Pack<T, V>*>(p);
    using Q = typename std::conditional<sizeof(T) == 4, quad_4, quad_2>::type;
    const Q q = __builtin_nontemporal_load(reinterpret_cast<const Q*>(p));
    Pack<T, V> out;
    __builtin_memcpy(&out, &q, sizeof(out) < 16 ? sizeof(out) : 16);
    return out;
}

template <typename TT, int V, bool NT = false>
__device__ __forceinline__ void store_row(TT* p, const float (&x)[V])
{
    Pack<TT, V> out;
#pragma unroll
    for (int v = 0; v < V; ++v) store_f32(out.v + v, x[v]);
    if (NT && sizeof(out) == 16) {
        using Q = typename std::conditional<sizeof(TT) == 4, quad_4, quad_2>::type;
        Q q;
        __builtin_memcpy(&q, &out, sizeof(out) < 16 ? sizeof(out) : 16);
        __builtin_nontemporal_store(q, reinterpret_cast<Q*>(p));
    } else {
        *reinterpret_cast<Pack<TT, V>*>(p) = out;
    }
}

__device__ __forceinline__ void zero_fill(char* p, long bytes, long at, long step)
{
    if (((uintptr_t)p & 15) == 0) {
        const long n = bytes >> 4;
        for (long i = at; i < n; i += step) nt_store4(make_float4(0.f, 0.f, 0.f, 0.f), reinterpret_cast<float4*>(p) + i);
        for (long i = (n << 4) + 2 * at; i < bytes; i += 2 * step) *reinterpret_cast<uint16_t*>(p + i) = 0;
    } else {
        for (long i = 2 * at; i < bytes; i += 2 * step) *reinterpret_cast<uint16_t*>(p + i) = 0;
    }
}

// the row of entry i, or -1
__device__ __forceinline__ long row_of(const LookupArgs& a, long i)
{
    const long id = a.ids_64 ? (long)reinterpret_cast<const int64_t*>(a.ids)[i] : (long)reinterpret_cast<const int32_t*>(a.ids)[i];
    return id >= 0 && id < a.rows ? id : -1;
}

// A group of G lanes per entry, V columns (16 bytes of the result) per lane; a wave takes 64 / G entries that follow one another at a
// time, so that its stores are one contiguous piece, and FWD_ENTRIES of them, so that as many gathers are in flight.
// NT: stores past the caches' normal replacement, for results larger than all L2s together: rows of 180 bytes begin and end inside a
// line, and lines that wait in the L2 for their other part crowd out what is being gathered (2 M rows of 45 floats: 121 us without,
// 67 with, 5.6 TB/s).  Smaller results are left in the caches for who reads them next.
constexpr int FWD_ENTRIES = 4;
constexpr long FWD_NT_BYTES = 32l << 20;

template <typename TT, typename TO, int V, bool NT>
__global__ void __launch_bounds__(256) k_lookup_fwd(LookupArgs a, TO* __restrict__ out, int g_shift)
{
    const int G = 1 << g_shift, lane = threadIdx.x & (G - 1), per = 64 >> g_shift;
    const long want = ((long)blockIdx.y * G + lane) * V;
    if (want >= a.width) return;
    // the last lane of a row that is no multiple of V starts early and writes some of its neighbour's columns again
    const long col = want + V <= a.width ? want : (a.width >= V ? a.width - V : 0);
    const long wave = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long first = wave * (per * FWD_ENTRIES) + ((threadIdx.x & 63) >> g_shift);
    const TT* table = reinterpret_cast<const TT*>(a.table) + col;
    long row[FWD_ENTRIES];
    float s[FWD_ENTRIES];
#pragma unroll
    for (int x = 0; x < FWD_ENTRIES; ++x) {
        const long i = first + x * per;
        row[x] = i < a.n ? row_of(a, i) : -1;
        s[x] = i < a.n && a.row_scale ? a.row_scale[i] : 1.0f;
    }
    Pack<TT, V> t[FWD_ENTRIES];
#pragma unroll
    for (int x = 0; x < FWD_ENTRIES; ++x)
        if (row[x] >= 0) t[x] = *reinterpret_cast<const Pack<TT, V>*>(table + row[x] * a.table_stride);
#pragma unroll
    for (int x = 0; x < FWD_ENTRIES; ++x) {
        const long i = first + x * per;
        if (i >= a.n) return;
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = row[x] >= 0 ? a.scale * s[x] * load_f32(t[x].v + v) : 0.0f;
        store_row<TO, V, NT>(out + i * a.width + col, y);
    }
}

// First launch of the table's gradient: the sort's keys -- the row, or `rows` for "no row" (sorted behind every row) -- and its values,
// the entries; workgroups behind those clear the gradient, of which only the rows with entries are written later.
__global__ void __launch_bounds__(256)
k_lookup_keys(LookupArgs a, uint32_t* __restrict__ key, uint32_t* __restrict__ val, int key_blocks, char* __restrict__ zero,
              long zero_bytes)
{
    if ((int)blockIdx.x < key_blocks) {
        const long i = (long)blockIdx.x * 256 + threadIdx.x;
        if (i >= a.n) return;
        const long row = row_of(a, i);
        key[i] = row >= 0 ? (uint32_t)row : (uint32_t)a.rows;
        val[i] = (uint32_t)i;
        return;
    }
    zero_fill(zero, zero_bytes, (long)(blockIdx.x - key_blocks) * 256 + threadIdx.x, (long)(gridDim.x - key_blocks) * 256);
}

constexpr uint32_t NO_ENTRY = 0xffffffffu;            // behind every row and behind "no row"

// ---- the sort of few entries by one workgroup: all of them stay in LDS through the passes (stable, 8 bits each).
constexpr int SORT_SMALL = 16384, SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;

template <int ITEMS>
struct SortLds {
    uint32_t cnt[SORT_WAVES][256], base[256], wave_sum[4];
    uint32_t key[SORT_THREADS * ITEMS], val[SORT_THREADS * ITEMS];
};

// Entries 0 .. n - 1 by their row (`rows` for "no row", padding behind it) into lds.key / lds.val.  All SORT_THREADS threads; the
// arrays may be read when it returns.
template <int ITEMS>
__device__ __forceinline__ void sort_entries(const LookupArgs& a, int bits, SortLds<ITEMS>& lds)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, first = w * (64 * ITEMS) + lane;
    const unsigned long long before = (1ull << lane) - 1ull;
    uint32_t key[ITEMS], val[ITEMS], rank[ITEMS];
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
        const int i = first + 64 * x;
        const long row = i < a.n ? row_of(a, i) : -1;
        key[x] = i < a.n ? (row >= 0 ? (uint32_t)row : (uint32_t)a.rows) : NO_ENTRY;
        val[x] = (uint32_t)i;
    }
    for (int shift = 0; shift < bits; shift += 8) {
        for (int d = threadIdx.x; d < SORT_WAVES * 256; d += SORT_THREADS) (&lds.cnt[0][0])[d] = 0;
        __syncthreads();
        // the entry's place among those of its digit in its wave: lanes of the same digit by ballots, earlier items from the count
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            const uint32_t d = (key[x] >> shift) & 255u;
            unsigned long long same = ~0ull;
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const unsigned long long on = __ballot((d >> b) & 1u);
                same &= ((d >> b) & 1u) ? on : ~on;
            }
            const uint32_t prior = lds.cnt[w][d];
            rank[x] = prior + (uint32_t)__popcll(same & before);
            __builtin_amdgcn_wave_barrier();
            if ((same & before) == 0) lds.cnt[w][d] = prior + (uint32_t)__popcll(same);
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        // exclusive sums over (digit, wave)
        uint32_t total = 0, incl = 0;
        if (threadIdx.x < 256) {
            for (int k = 0; k < SORT_WAVES; ++k) {
                const uint32_t c = lds.cnt[k][threadIdx.x];
                lds.cnt[k][threadIdx.x] = total;
                total += c;
            }
            incl = total;
#pragma unroll
            for (int dd = 1; dd < 64; dd <<= 1) {
                const uint32_t o = (uint32_t)__shfl_up((int)incl, dd, 64);
                if (lane >= dd) incl += o;
            }
            if (lane == 63) lds.wave_sum[w] = incl;
        }
        __syncthreads();
        if (threadIdx.x < 256) {
            uint32_t b = incl - total;
            for (int k = 0; k < w; ++k) b += lds.wave_sum[k];
            lds.base[threadIdx.x] = b;
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            const uint32_t d = (key[x] >> shift) & 255u, at = lds.base[d] + lds.cnt[w][d] + rank[x];
            lds.key[at] = key[x];
            lds.val[at] = val[x];
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            key[x] = lds.key[first + 64 * x];
            val[x] = lds.val[first + 64 * x];
        }
    }
}

// First launch for up to SORT_SMALL entries: one workgroup sorts, the others clear the gradient meanwhile.  (The general sort takes a
// launch for the keys and four a pass: at 16384 entries and 32000 rows 49 us of kernels, and as much again between them; this one 35.)
template <int ITEMS>
__global__ void __launch_bounds__(SORT_THREADS)
k_lookup_sort(LookupArgs a, uint32_t* __restrict__ key_out, uint32_t* __restrict__ val_out, int bits, char* __restrict__ zero, long zero_bytes)
{
    __shared__ SortLds<ITEMS> lds;
    if (blockIdx.x > 0) {
        zero_fill(zero, zero_bytes, (long)(blockIdx.x - 1) * SORT_THREADS + threadIdx.x, (long)(gridDim.x - 1) * SORT_THREADS);
        return;
    }
    sort_entries<ITEMS>(a, bits, lds);
    for (int i = threadIdx.x; i < a.n; i += SORT_THREADS) {
        key_out[i] = lds.key[i];
        val_out[i] = lds.val[i];
    }
}

// ---- the sums of the table's gradient over the sorted entries.
//
// Split by ENTRIES, not by rows, so that a row hit a million times costs what a million rows hit once do: a group of G lanes
// (V columns each; G x V covers the width, or a tile of it) takes a chunk of consecutive sorted entries, keeps the running sum of the
// current row in registers and stores it where the row changes.  A row that begins and ends inside the chunk goes straight to the
// gradient; the sum of one that crosses the chunk's border goes to a slot of its own -- head: of the row that came in from the chunk
// before; tail: of the row that begins here and goes on -- and k_lookup_join adds a row's tail and the heads behind it in order.
// No atomics, and every order fixed by n and width alone.
//
// The gradient rows are gathered: each is one contiguous read of width x 4 bytes, UNROLL of them in flight per lane.
constexpr int UNROLL = 8;

struct SumArgs {
    const uint32_t *key, *val;
    const void* grad;
    long grad_stride;
    void* d_table;
    float* d_row_scale;
    float* slots;                 // [chunks][2][width]: head, tail
    int chunk;                    // entries of a chunk, a multiple of UNROLL
    int g_shift;                  // G = 1 << g_shift lanes
};

template <typename TT, typename TO, int V, bool DSCALE>
__global__ void __launch_bounds__(256) k_lookup_sum(LookupArgs a, SumArgs q)
{
    const int G = 1 << q.g_shift, lane = threadIdx.x & (G - 1);
    const long chunk = ((long)blockIdx.x * 256 + threadIdx.x) >> q.g_shift;
    const long first = chunk * q.chunk, last = first + q.chunk < a.n ? first + q.chunk : a.n;
    // the last lane of a row that is no multiple of V starts early and computes some of its neighbour's columns again
    const long want = ((long)blockIdx.y * G + lane) * V;
    const bool live = first < a.n && want < a.width;
    const long col = want + V <= a.width ? want : (a.width >= V ? a.width - V : 0);
    if (first >= a.n) return;               // (whole groups: the shuffles below stay inside a group)
    const uint32_t rows = (uint32_t)a.rows;
    const TO* grad = reinterpret_cast<const TO*>(q.grad) + col;
    const TT* table = reinterpret_cast<const TT*>(a.table) + col;
    TT* d_table = reinterpret_cast<TT*>(q.d_table) + col;
    float* slot = q.slots + (2 * chunk) * a.width + col;
    // (the arrays are padded to whole chunks: the loads of keys and entries need no bounds, what lies behind `last` is masked)
    uint4 next_key[UNROLL / 4], next_val[UNROLL / 4];
#pragma unroll
    for (int x = 0; x < UNROLL / 4; ++x) {
        next_key[x] = reinterpret_cast<const uint4*>(q.key + first)[x];
        next_val[x] = reinterpret_cast<const uint4*>(q.val + first)[x];
    }
    uint32_t cur = q.key[first];
    bool came_in = first > 0 && q.key[first - 1] == cur;
    float acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.0f;
    for (long j = first; j < last; j += UNROLL) {
        uint32_t key[UNROLL], val[UNROLL];
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) {
            const bool in = j + x < last;
            key[x] = in ? (&next_key[x / 4].x)[x % 4] : NO_ENTRY;
            val[x] = in ? (&next_val[x / 4].x)[x % 4] : 0u;
        }
        Pack<TO, V> g[UNROLL];
        Pack<TT, V> t[UNROLL];
        float s[UNROLL];
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) {
            const bool there = key[x] < rows;
            s[x] = there && a.row_scale ? a.row_scale[val[x]] : 1.0f;
            g[x] = load_once<TO, V>(grad + (there ? (long)val[x] * q.grad_stride : 0));
            if (DSCALE) t[x] = *reinterpret_cast<const Pack<TT, V>*>(table + (there ? (long)key[x] * a.table_stride : 0));
        }
        if (j + UNROLL < last) {               // the next ones travel while these rows are added
#pragma unroll
            for (int x = 0; x < UNROLL / 4; ++x) {
                next_key[x] = reinterpret_cast<const uint4*>(q.key + j + UNROLL)[x];
                next_val[x] = reinterpret_cast<const uint4*>(q.val + j + UNROLL)[x];
            }
        }
        float dot[UNROLL];
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) {
            if (key[x] != cur && key[x] != NO_ENTRY) {
                if (live && cur < rows) {
                    if (came_in) store_row<float, V>(slot, acc);
                    else store_row<TT, V>(d_table + (long)cur * a.width, acc);
                }
                came_in = false;
                cur = key[x];
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] = 0.0f;
            }
            dot[x] = 0.0f;
            if (key[x] < rows) {
                const float sx = a.scale * s[x];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float gv = load_f32(g[x].v + v);
                    acc[v] = fmaf(sx, gv, acc[v]);
                    if (DSCALE && col + v >= want) dot[x] = fmaf(gv, load_f32(t[x].v + v), dot[x]);
                }
            }
        }
        if (DSCALE) {
#pragma unroll
            for (int x = 0; x < UNROLL; ++x) {
                float d = live ? dot[x] : 0.0f;
                for (int w = G >> 1; w > 0; w >>= 1) d += __shfl_xor(d, w, 64);
                if (lane == 0 && j + x < last) q.d_row_scale[val[x]] = a.scale * d;
            }
        }
    }
    if (live && cur < rows) {
        const bool goes_on = last < a.n && q.key[last] == cur;
        if (came_in) store_row<float, V>(slot, acc);
        else if (goes_on) store_row<float, V>(slot + a.width, acc);
        else store_row<TT, V>(d_table + (long)cur * a.width, acc);
    }
}

// Rows that cross borders of chunks: tail[c] + head[c + 1] + ... + head[end].  A workgroup looks at JOIN_CHUNKS chunks; short
// rows are one group's each, rows of more than JOIN_LONG pieces the whole workgroup's: group k adds the pieces k, k + groups, ... and
// the groups' sums are added in order.
constexpr int JOIN_THREADS = 1024, JOIN_CHUNKS = 64, JOIN_LONG = 16, JOIN_AHEAD = 8;

// acc += the pieces p, p + step, ... up to `end` of the row whose tail is piece c, JOIN_AHEAD of them in flight
template <int V>
__device__ __forceinline__ void join_pieces(float (&acc)[V], const float* __restrict__ slots, long width, long c, long p, long end,
                                            long step)
{
    for (; p <= end; p += JOIN_AHEAD * step) {
        Pack<float, V> h[JOIN_AHEAD];
#pragma unroll
        for (int x = 0; x < JOIN_AHEAD; ++x) {
            const long at = p + x * step <= end ? p + x * step : p;
            h[x] = *reinterpret_cast<const Pack<float, V>*>(slots + (2 * at + (at == c)) * width);
        }
#pragma unroll
        for (int x = 0; x < JOIN_AHEAD; ++x)
            if (p + x * step <= end)
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] += h[x].v[v];
    }
}

template <typename TT, int V>
__global__ void __launch_bounds__(JOIN_THREADS) k_lookup_join(LookupArgs a, SumArgs q, long chunks)
{
    __shared__ long from[JOIN_CHUNKS], upto[JOIN_CHUNKS];
    __shared__ uint32_t row[JOIN_CHUNKS];
    __shared__ int count;
    __shared__ float part[JOIN_THREADS * V];
    const int G = 1 << q.g_shift, lane = threadIdx.x & (G - 1), group = threadIdx.x >> q.g_shift, groups = JOIN_THREADS >> q.g_shift;
    const long want = ((long)blockIdx.y * G + lane) * V;
    const bool live = want < a.width;
    const long col = want + V <= a.width ? want : (a.width >= V ? a.width - V : 0);
    if (threadIdx.x < JOIN_CHUNKS) {
        const long c = (long)blockIdx.x * JOIN_CHUNKS + threadIdx.x, first = c * q.chunk, next = first + q.chunk;
        bool owner = false;
        uint32_t k = 0;
        if (c < chunks && next < a.n) {
            k = q.key[next - 1];
            // its last row goes on, and begins in this chunk
            owner = k < (uint32_t)a.rows && q.key[next] == k && (first == 0 || q.key[first - 1] != k);
        }
        const unsigned long long mask = __ballot(owner);           // (one wave: JOIN_CHUNKS is 64)
        if (threadIdx.x == 0) count = __popcll(mask);
        if (owner) {
            // the last chunk whose first entry is of this row: doubling steps, then halving ones
            long lo = c + 1, step = 1;
            while (lo + step < chunks && q.key[(lo + step) * q.chunk] == k) { lo += step; step <<= 1; }
            for (; step > 0; step >>= 1)
                if (lo + step < chunks && q.key[(lo + step) * q.chunk] == k) lo += step;
            const int at = __popcll(mask & ((1ull << threadIdx.x) - 1ull));
            from[at] = c; upto[at] = lo; row[at] = k;
        }
    }
    __syncthreads();
    const float* slots = q.slots + col;
    TT* d_table = reinterpret_cast<TT*>(q.d_table) + col;
    for (int o = group; o < count; o += groups) {
        const long c = from[o], end = upto[o];
        if (end - c > JOIN_LONG || !live) continue;
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        join_pieces<V>(acc, slots, a.width, c, c, end, 1);
        store_row<TT, V>(d_table + (long)row[o] * a.width, acc);
    }
    for (int o = 0; o < count; ++o) {
        const long c = from[o], end = upto[o];
        if (end - c <= JOIN_LONG) continue;                         // (the same for every thread)
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        join_pieces<V>(acc, slots, a.width, c, c + group, end, groups);
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) part[threadIdx.x * V + v] = acc[v];
        __syncthreads();
        if (group == 0 && live) {
            for (int k = 1; k < groups; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] += part[((k << q.g_shift) + lane) * V + v];
            store_row<TT, V>(d_table + (long)row[o] * a.width, acc);
        }
    }
}

// ---- up to SMALL entries in one launch without any scratch: every workgroup sorts all of them in its LDS and writes the rows of its own
// range, the ones without entries as zeros.  A row is one group's; one of more than SMALL_LONG entries is the whole workgroup's, in
// contiguous pieces that are added in order.  (100 entries, 1000 rows of ten floats: 6 us against 12 for the three launches.)
constexpr int SMALL = SORT_THREADS, SMALL_LONG = 32;

__device__ __forceinline__ int first_at_least(const uint32_t* key, int n, uint32_t k)
{
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (key[mid] < k) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// acc += the entries j .. end - 1, all of the row at `table`
template <typename TT, typename TO, int V, bool DSCALE>
__device__ __forceinline__ void add_entries(const LookupArgs& a, const SumArgs& q, const uint32_t* val, int j, int end, long col, long want,
                                            bool live, const TT* table, float (&acc)[V])
{
    const TO* grad = reinterpret_cast<const TO*>(q.grad) + col;
    const int G = 1 << q.g_shift, lane = threadIdx.x & (G - 1);
    Pack<TT, V> t;
    if (DSCALE) t = *reinterpret_cast<const Pack<TT, V>*>(table);
    for (; j < end; j += UNROLL) {
        Pack<TO, V> g[UNROLL];
        float s[UNROLL];
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) {
            const long i = val[j + x < end ? j + x : j];
            s[x] = a.row_scale ? a.row_scale[i] : 1.0f;
            g[x] = load_once<TO, V>(grad + i * q.grad_stride);
        }
#pragma unroll
        for (int x = 0; x < UNROLL; ++x) {
            if (j + x >= end) break;
            const float sx = a.scale * s[x];
            float dot = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float gv = load_f32(g[x].v + v);
                acc[v] = fmaf(sx, gv, acc[v]);
                if (DSCALE && live && col + v >= want) dot = fmaf(gv, load_f32(t.v + v), dot);
            }
            if (DSCALE) {
                for (int w = G >> 1; w > 0; w >>= 1) dot += __shfl_xor(dot, w, 64);
                if (lane == 0) q.d_row_scale[val[j + x]] = a.scale * dot;
            }
        }
    }
}

template <typename TT, typename TO, int V, bool DSCALE>
__global__ void __launch_bounds__(SORT_THREADS) k_lookup_small(LookupArgs a, SumArgs q, int bits, long rows_each)
{
    __shared__ SortLds<1> lds;
    __shared__ float part[SORT_THREADS * V];
    __shared__ int long_runs[SMALL / SMALL_LONG], n_long;
    if (threadIdx.x == 0) n_long = 0;
    sort_entries<1>(a, bits, lds);
    const int n = (int)a.n, G = 1 << q.g_shift, lane = threadIdx.x & (G - 1), group = threadIdx.x >> q.g_shift, groups = SORT_THREADS >> q.g_shift;
    const long r0 = (long)blockIdx.x * rows_each, r1 = r0 + rows_each < a.rows ? r0 + rows_each : a.rows;
    const long want = ((long)blockIdx.y * G + lane) * V;
    const bool live = want < a.width;
    const long col = want + V <= a.width ? want : (a.width >= V ? a.width - V : 0);
    const TT* table = reinterpret_cast<const TT*>(a.table) + col;
    TT* d_table = reinterpret_cast<TT*>(q.d_table) + col;
    const int e0 = first_at_least(lds.key, n, (uint32_t)r0), e1 = first_at_least(lds.key, n, (uint32_t)r1);
    float acc[V];
    // rows without entries
    for (long r = r0 + group; r < r1; r += groups) {
        const int at = first_at_least(lds.key, n, (uint32_t)r);
        if (live && (at >= n || lds.key[at] != (uint32_t)r)) {
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = 0.0f;
            store_row<TT, V>(d_table + r * a.width, acc);
        }
    }
    if (DSCALE && blockIdx.x == 0)                               // entries without a row
        for (int j = threadIdx.x; j < n; j += SORT_THREADS)
            if (lds.key[j] >= (uint32_t)a.rows) q.d_row_scale[lds.val[j]] = 0.0f;
    // rows with entries: the group of the row's first one
    for (int j = e0 + group; j < e1; j += groups) {
        const uint32_t k = lds.key[j];
        if (j > e0 && lds.key[j - 1] == k) continue;
        const int end = first_at_least(lds.key, n, k + 1);
        if (end - j > SMALL_LONG) {
            if (lane == 0) long_runs[atomicAdd(&n_long, 1)] = j;       // (their order does not matter: each is a row of its own)
            continue;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        add_entries<TT, TO, V, DSCALE>(a, q, lds.val, j, end, col, want, live, table + (long)k * a.table_stride, acc);
        if (live) store_row<TT, V>(d_table + (long)k * a.width, acc);
    }
    __syncthreads();
    for (int o = 0; o < n_long; ++o) {
        const int j = long_runs[o];
        const uint32_t k = lds.key[j];
        const int end = first_at_least(lds.key, n, k + 1), each = (end - j + groups - 1) / groups;
        const int from = j + group * each, upto = from + each < end ? from + each : end;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        if (from < upto) add_entries<TT, TO, V, DSCALE>(a, q, lds.val, from, upto, col, want, live, table + (long)k * a.table_stride, acc);
#pragma unroll
        for (int v = 0; v < V; ++v) part[threadIdx.x * V + v] = acc[v];
        __syncthreads();
        if (group == 0 && live) {
            for (int g = 1; g < groups && g * each < end - j; ++g)
#pragma unroll
                for (int v = 0; v < V; ++v) acc[v] += part[((g << q.g_shift) + lane) * V + v];
            store_row<TT, V>(d_table + (long)k * a.width, acc);
        }
        __syncthreads();
    }
}

// The scales' gradient alone, entry by entry: where the table's is not wanted, or the width takes more than one tile.
template <typename TT, typename TO, int V>
__global__ void __launch_bounds__(256) k_lookup_dscale(LookupArgs a, const TO* __restrict__ grad, long grad_stride,
                                                       float* __restrict__ d_row_scale, int g_shift)
{
    const int G = 1 << g_shift, lane = threadIdx.x & (G - 1);
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) >> g_shift;
    if (i >= a.n) return;
    const long row = row_of(a, i);
    float acc = 0.0f;
    if (row >= 0) {
        const TO* g = grad + i * grad_stride;
        const TT* t = reinterpret_cast<const TT*>(a.table) + row * a.table_stride;
        for (long want = (long)lane * V; want < a.width; want += G * V) {
            const long col = want + V <= a.width ? want : (a.width >= V ? a.width - V : 0);
            const Pack<TO, V> x = *reinterpret_cast<const Pack<TO, V>*>(g + col);
            const Pack<TT, V> y = *reinterpret_cast<const Pack<TT, V>*>(t + col);
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (col + v >= want) acc = fmaf(load_f32(x.v + v), load_f32(y.v + v), acc);
        }
    }
    for (int w = G >> 1; w > 0; w >>= 1) acc += __shfl_xor(acc, w, 64);
    if (lane == 0) d_row_scale[i] = a.scale * acc;
}

// Lanes and columns for a width: V values (16 bytes of the result's type) per lane, or one where the row is shorter than that.
struct Tiling {
    int V, g_shift, tiles, chunk;
    long chunks;
};
static Tiling tiling(int64_t n, int64_t width, int v_full)
{
    Tiling t;
    t.V = width >= v_full ? v_full : 1;
    const int64_t lanes = (width + t.V - 1) / t.V;
    t.g_shift = 0;
    while (t.g_shift < 6 && (1 << t.g_shift) < lanes) ++t.g_shift;
    t.tiles = (int)((lanes + 63) / 64);
    // long chunks make few slots; shorter ones while there are fewer than four waves for each of the 1024 SIMDs -- but no more than
    // 8192 of them, which is what one workgroup has to join where all entries are of one row (at 16384 entries of 1024 16-bit
    // values: 13 us with four waves per SIMD, 19 with one)
    t.chunk = 64;
    while (t.chunk > UNROLL && ((n << t.g_shift) / 64 / t.chunk) * t.tiles < 4096 && n <= 4096l * t.chunk) t.chunk >>= 1;
    t.chunks = (long)((n + t.chunk - 1) / t.chunk);
    return t;
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
        constexpr int V = 16 / sizeof(TO);
        const Tiling t = tiling(a.n, a.width, V);
        const long per = 4 * (64 >> t.g_shift) * FWD_ENTRIES;
        const dim3 grid((unsigned)((a.n + per - 1) / per), t.tiles);
        if (t.V != V) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_fwd<TT, TO, 1, false>), grid, dim3(256), 0, s, a, (TO*)out, t.g_shift);
        else if (a.n * a.width * (long)sizeof(TO) >= FWD_NT_BYTES)
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_fwd<TT, TO, V, true>), grid, dim3(256), 0, s, a, (TO*)out, t.g_shift);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_fwd<TT, TO, V, false>), grid, dim3(256), 0, s, a, (TO*)out, t.g_shift);
        if (hipGetLastError() != hipSuccess) { set_error("lookup: kernel launch failed"); return VR_ERR_HIP; }
        return VR_OK;
    }
};

// Everything after the sort.
struct Backward {
    template <typename TT, typename TO, int V>
    static void launch(const LookupArgs& a, const SumArgs& q, const Tiling& t, hipStream_t s)
    {
        const bool fused = q.d_row_scale && q.d_table && t.tiles == 1;
        if (q.d_table && a.n <= SMALL) {
            // (a row's columns may take several workgroups: 256 ranges of rows, or fewer)
            const long rows_each = (a.rows + 255) / 256;
            const dim3 grid((unsigned)((a.rows + rows_each - 1) / rows_each), t.tiles);
            if (fused) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_small<TT, TO, V, true>), grid, dim3(SORT_THREADS), 0, s, a, q, key_bits(a.rows), rows_each);
            else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_small<TT, TO, V, false>), grid, dim3(SORT_THREADS), 0, s, a, q, key_bits(a.rows), rows_each);
        } else if (q.d_table) {
            const dim3 grid((unsigned)(((t.chunks << t.g_shift) + 255) / 256), t.tiles);
            if (fused) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_sum<TT, TO, V, true>), grid, dim3(256), 0, s, a, q);
            else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_sum<TT, TO, V, false>), grid, dim3(256), 0, s, a, q);
            if (t.chunks > 1)
                hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_join<TT, V>), dim3((unsigned)((t.chunks + JOIN_CHUNKS - 1) / JOIN_CHUNKS), t.tiles),
                                   dim3(JOIN_THREADS), 0, s, a, q, t.chunks);
        }
        if (q.d_row_scale && !fused)
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_dscale<TT, TO, V>), dim3((unsigned)(((a.n << t.g_shift) + 255) / 256)), dim3(256),
                               0, s, a, reinterpret_cast<const TO*>(q.grad), q.grad_stride, q.d_row_scale, t.g_shift);
    }
    template <typename TT, typename TO>
    static int run(const LookupArgs& a, SumArgs q, hipStream_t s)
    {
        constexpr int V = 16 / sizeof(TO);
        const Tiling t = tiling(a.n, a.width, V);
        q.chunk = t.chunk;
        q.g_shift = t.g_shift;
        if (t.V == V) launch<TT, TO, V>(a, q, t, s);
        else launch<TT, TO, 1>(a, q, t, s);
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

// scratch: two pairs of key and value arrays, the sort's own, and the slots of the chunks (a chunk has UNROLL entries at
// least; the tiling of the wider type has the shorter chunks)
static size_t slots_bytes(int64_t n, int64_t width)
{
    const long chunks = tiling(n, width, 4).chunks > tiling(n, width, 8).chunks ? tiling(n, width, 4).chunks : tiling(n, width, 8).chunks;
    return align_up((size_t)chunks * 2 * (size_t)width * sizeof(float), 256);
}

extern "C" int64_t vr_lookup_scratch_bytes(int64_t n, int64_t rows, int64_t width)
{
    if (n < 0 || n >= (1ll << 30) || rows < 0 || rows >= 0x7fffffffll || width < 1 || width > (1 << 24)) return 0;
    if (n <= SMALL) return 0;
    return (int64_t)(4 * align_up((size_t)n * 4, 256) + align_up(sort_pairs_scratch_bytes((long)n), 256) + slots_bytes(n, width));
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
    if (d_table && a.n > SMALL && (!scratch || ((uintptr_t)scratch & 255) || scratch_bytes < vr_lookup_scratch_bytes(a.n, a.rows, a.width)))
        { set_error("lookup: the table's gradient needs vr_lookup_scratch_bytes of scratch, 256-byte aligned"); return VR_ERR_INVALID_ARGUMENT; }
    if (a.rows == 0) d_table = nullptr;
    if (!d_table && (!d_row_scale || a.n == 0)) return VR_OK;
    hipStream_t s = (hipStream_t)stream;
    SumArgs q{nullptr, nullptr, grad, (long)grad_stride, d_table, d_row_scale, nullptr, 0, 0};
    if (d_table && a.n > SMALL) {
        const size_t arr = align_up((size_t)a.n * 4, 256);
        char* base = (char*)scratch;
        uint32_t *k0 = (uint32_t*)base, *v0 = (uint32_t*)(base + arr), *k1 = (uint32_t*)(base + 2 * arr), *v1 = (uint32_t*)(base + 3 * arr);
        const long zero_bytes = a.rows * a.width * (long)t_element, zero_blocks = (zero_bytes + 16383) / 16384;
        if (a.n <= SORT_SMALL) {
            const dim3 grid(1 + (unsigned)(zero_blocks < 1024 ? zero_blocks : 1024));
            const int bits = key_bits(a.rows);
            if (a.n <= 4 * SORT_THREADS) hipLaunchKernelGGL(k_lookup_sort<4>, grid, dim3(SORT_THREADS), 0, s, a, k0, v0, bits, (char*)d_table, zero_bytes);
            else hipLaunchKernelGGL(k_lookup_sort<16>, grid, dim3(SORT_THREADS), 0, s, a, k0, v0, bits, (char*)d_table, zero_bytes);
            VR_KERNEL_CHECK("lookup_sort", s, false);
            q.key = k0;
            q.val = v0;
        } else {
            const int key_blocks = cdiv(a.n, 256);
            hipLaunchKernelGGL(k_lookup_keys, dim3(key_blocks + (unsigned)(zero_blocks < 4096 ? zero_blocks : 4096)), dim3(256), 0, s, a, k0,
                               v0, key_blocks, (char*)d_table, zero_bytes);
            VR_KERNEL_CHECK("lookup_keys", s, false);
            int where = 0;
            if (int rc = launch_sort_pairs(k0, v0, k1, v1, a.n, 0u, key_bits(a.rows), base + 4 * arr, s, false, &where)) return rc;
            q.key = where ? k1 : k0;
            q.val = where ? v1 : v0;
        }
        q.slots = (float*)(base + 4 * arr + align_up(sort_pairs_scratch_bytes(a.n), 256));
    }
    return by_type<Backward>(lookup, a, q, s);
}
