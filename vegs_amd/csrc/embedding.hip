// embedding.hip -- the row lookup and its gradients (include/vegs_embedding.h).
//
//   out[i] = s_i T[id_i]        dT[k] = sum_{i: id_i = k} s_i g_i        ds_i = <g_i, T[id_i]>
//
// Bound by memory: two operations per value.  Forward, the table is read from the caches and the result written once, streamed.
// Backward, every gradient row is read once, in the order of the rows of T it goes to (a stable sort of the ids), so that a row's sum is
// formed in registers without atomics, in an order that the sizes and the ids fix.  Measured at 2 M entries of 45 floats, 8192
// rows: forward 65 us (5.8 TB/s); sort 53, sums with the scales' gradient 141 (the rows of 180 bytes come as whole lines: 600 MB for their
// 360), join 12.  Short inputs are bound by launches: up to 1024 entries take one, up to 16384 three.
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

// 16 bytes at an address of 2 or 4 bytes' alignment; ONCE: past the caches' normal order of replacement
typedef uint32_t quad_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t quad_2 __attribute__((ext_vector_type(4), aligned(2)));

template <typename T, int V, bool ONCE>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p)
{
    if (!ONCE || sizeof(Pack<T, V>) != 16) return *reinterpret_cast<const Pack<T, V>*>(p);
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
    const long wave = ((long)blockIdx.z * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
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

constexpr uint32_t NO_ENTRY = 0xffffffffu;            // behind every row and behind "no row"

// between a wave's reads and writes of the same LDS words: the hardware keeps a wave's LDS operations in order, this the compiler's
__device__ __forceinline__ void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- the sort of few entries inside a workgroup: they stay in LDS through the passes (stable, digits of up to 8 bits).
constexpr int SORT_SMALL = 16384, SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64, SORT_GROUPS = 16;

template <int ITEMS>
struct SortLds {
    uint32_t cnt[SORT_WAVES][256], base[256], wave_sum[4];
    uint32_t key[SORT_THREADS * ITEMS], val[SORT_THREADS * ITEMS];
};

// lds.key / lds.val [0, m), keys of `bits` bits from `lo` on, into ascending order.  All SORT_THREADS threads; the arrays have been
// written and synchronised before, and may be read by everyone after.
template <int ITEMS>
__device__ __forceinline__ void sort_in_lds(SortLds<ITEMS>& lds, int m, uint32_t lo, int bits)
{
    const int items = (m + SORT_THREADS - 1) / SORT_THREADS;                  // of each thread; what they are more than m stays last
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, first = w * (64 * items) + lane;
    const unsigned long long before = (1ull << lane) - 1ull;
    uint32_t key[ITEMS], val[ITEMS], rank[ITEMS];
    for (int shift = 0; shift < bits; shift += 8) {
        const int digit_bits = bits - shift < 8 ? bits - shift : 8;
        const uint32_t mask = (1u << digit_bits) - 1u;
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            if (x < items) {
                key[x] = lds.key[first + 64 * x];
                val[x] = lds.val[first + 64 * x];
            }
        }
        for (int d = threadIdx.x; d < SORT_WAVES * 256; d += SORT_THREADS) (&lds.cnt[0][0])[d] = 0;
        __syncthreads();
        // the entry's place among those of its digit in its wave: lanes of the same digit by ballots, earlier items from the count
#pragma unroll
        for (int x = 0; x < ITEMS; ++x) {
            if (x >= items) continue;
            const uint32_t d = first + 64 * x < m ? ((key[x] - lo) >> shift) & mask : mask;
            unsigned long long same = ~0ull;
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                if (b >= digit_bits) continue;
                const unsigned long long on = __ballot((d >> b) & 1u);
                same &= ((d >> b) & 1u) ? on : ~on;
            }
            const uint32_t prior = lds.cnt[w][d];
            rank[x] = prior + (uint32_t)__popcll(same & before);
            wave_order();
            if ((same & before) == 0) lds.cnt[w][d] = prior + (uint32_t)__popcll(same);
            wave_order();
        }
        __syncthreads();
        // exclusive sums over (digit, wave)
        uint32_t total = 0, incl = 0;
        if (threadIdx.x < 256) {
#pragma unroll
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
            if (x >= items) continue;
            const uint32_t d = first + 64 * x < m ? ((key[x] - lo) >> shift) & mask : mask, at = lds.base[d] + lds.cnt[w][d] + rank[x];
            lds.key[at] = key[x];
            lds.val[at] = val[x];
        }
        __syncthreads();
    }
}

__device__ __forceinline__ uint32_t key_of(const LookupArgs& a, long i)
{
    const long row = row_of(a, i);
    return row >= 0 ? (uint32_t)row : (uint32_t)a.rows;
}

// First launch for up to SORT_SMALL entries.  SORT_GROUPS workgroups read all ids, take the entries of their own range of rows in order
// into LDS, sort them there and write them behind the entries of smaller rows, which they have counted; the workgroups behind them clear
// the gradient meanwhile.  (16384 entries of 32000 rows and 65 MB to clear: 40 us with one workgroup sorting all -- which is what it comes
// to where all are of one range --, 24 with these; the general sort below takes six launches of 30 us together.)
__global__ void __launch_bounds__(SORT_THREADS)
k_lookup_sort(LookupArgs a, uint32_t* __restrict__ key_out, uint32_t* __restrict__ val_out, uint32_t range, int bits, char* __restrict__ zero,
              long zero_bytes)
{
    constexpr int ITEMS = SORT_SMALL / SORT_THREADS;
    __shared__ SortLds<ITEMS> lds;
    __shared__ int in_range[SORT_WAVES], below[SORT_WAVES];
    if (blockIdx.x >= SORT_GROUPS) {
        zero_fill(zero, zero_bytes, (long)(blockIdx.x - SORT_GROUPS) * SORT_THREADS + threadIdx.x,
                  (long)(gridDim.x - SORT_GROUPS) * SORT_THREADS);
        return;
    }
    const int n = (int)a.n, items = (n + SORT_THREADS - 1) / SORT_THREADS;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, first = w * (64 * items) + lane;
    const unsigned long long before = (1ull << lane) - 1ull;
    const uint32_t lo = blockIdx.x * range;                        // (the last range holds "no row" too, or lies behind it)
    int mine = 0, smaller = 0;
    uint32_t key[ITEMS];
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
        if (x >= items) continue;
        const int i = first + 64 * x;
        key[x] = i < n ? key_of(a, i) : NO_ENTRY;
    }
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
        if (x >= items) continue;
        mine += __popcll(__ballot(key[x] >= lo && key[x] - lo < range && key[x] != NO_ENTRY));
        smaller += __popcll(__ballot(key[x] < lo));
    }
    if (lane == 0) { in_range[w] = mine; below[w] = smaller; }
    __syncthreads();
    int at = 0, m = 0, out = 0;
    for (int k = 0; k < SORT_WAVES; ++k) {
        at += k < w ? in_range[k] : 0;
        m += in_range[k];
        out += below[k];
    }
#pragma unroll
    for (int x = 0; x < ITEMS; ++x) {
        if (x >= items) continue;
        const bool in = key[x] >= lo && key[x] - lo < range && key[x] != NO_ENTRY;
        const unsigned long long on = __ballot(in);
        if (in) {
            const int to = at + __popcll(on & before);
            lds.key[to] = key[x];
            lds.val[to] = (uint32_t)(first + 64 * x);
        }
        at += __popcll(on);
    }
    __syncthreads();
    sort_in_lds<ITEMS>(lds, m, lo, bits);
    for (int i = threadIdx.x; i < m; i += SORT_THREADS) {
        key_out[out + i] = lds.key[i];
        val_out[out + i] = lds.val[i];
    }
}

// ---- the sort of many entries: stable, least significant digit first, digits of up to 8 bits; a pass is a histogram per block of
// SORT_BLOCK entries, the sums over the blocks of each digit, and the scatter.  The first pass takes its keys from the ids, and its
// histogram's launch clears the table's gradient in further workgroups.  The scales travel with the entries: gathered afterwards, every
// one of them would fetch a line of its own (2 M entries: the sums 7 us longer, the passes 1 each shorter).
constexpr int SORT_BLOCK = 4096, PASS_THREADS = 1024, PASS_WAVES = PASS_THREADS / 64, PASS_ITEMS = SORT_BLOCK / PASS_THREADS;

struct PassArgs {
    const uint32_t *key, *val;      // NULL in the first pass: from the ids
    const float* scale;             // NULL: none travel
    uint32_t *key_out, *val_out;
    float* scale_out;
    uint32_t *hist, *totals;        // [digits][blocks] counts, then their exclusive sums; [digits]
    int blocks, shift, bits;
};

__device__ __forceinline__ uint32_t pass_key(const LookupArgs& a, const PassArgs& p, long i)
{
    if (p.key) return p.key[i];
    return key_of(a, i);
}

__global__ void __launch_bounds__(PASS_THREADS) k_sort_hist(LookupArgs a, PassArgs p, char* __restrict__ zero, long zero_bytes)
{
    __shared__ uint32_t count[256];
    if ((int)blockIdx.x >= p.blocks) {
        zero_fill(zero, zero_bytes, (long)(blockIdx.x - p.blocks) * PASS_THREADS + threadIdx.x, (long)(gridDim.x - p.blocks) * PASS_THREADS);
        return;
    }
    const uint32_t mask = (1u << p.bits) - 1u;
    if (threadIdx.x < 256) count[threadIdx.x] = 0;
    __syncthreads();
    uint32_t key[PASS_ITEMS];
#pragma unroll
    for (int x = 0; x < PASS_ITEMS; ++x) {
        const long i = (long)blockIdx.x * SORT_BLOCK + x * PASS_THREADS + threadIdx.x;
        key[x] = i < a.n ? pass_key(a, p, i) : 0u;
    }
#pragma unroll
    for (int x = 0; x < PASS_ITEMS; ++x) {
        const long i = (long)blockIdx.x * SORT_BLOCK + x * PASS_THREADS + threadIdx.x;
        if (i < a.n) atomicAdd(&count[(key[x] >> p.shift) & mask], 1u);        // (counts: their order does not matter)
    }
    __syncthreads();
    if (threadIdx.x <= mask) p.hist[(size_t)threadIdx.x * p.blocks + blockIdx.x] = count[threadIdx.x];
}

// one workgroup per digit: the exclusive sums of its counts over the blocks, in place, and their total
__global__ void __launch_bounds__(256) k_sort_sums(PassArgs p)
{
    __shared__ uint32_t wave_sum[4];
    uint32_t* h = p.hist + (size_t)blockIdx.x * p.blocks;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int first = 0; first < p.blocks; first += 256) {
        const int i = first + threadIdx.x;
        const uint32_t c = i < p.blocks ? h[i] : 0u;
        uint32_t incl = c;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)incl, d, 64);
            if (lane >= d) incl += o;
        }
        if (lane == 63) wave_sum[w] = incl;
        __syncthreads();
        uint32_t base = carry;
        for (int k = 0; k < w; ++k) base += wave_sum[k];
        if (i < p.blocks) h[i] = base + incl - c;
        carry += wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) p.totals[blockIdx.x] = carry;
}

// The block's entries are put in the order of their digits in LDS first, so that what goes to one digit leaves as one piece.
__global__ void __launch_bounds__(PASS_THREADS) k_sort_scatter(LookupArgs a, PassArgs p)
{
    __shared__ uint32_t cnt[PASS_WAVES][256], local[256], global[256], wave_sum[2][4];
    __shared__ uint32_t skey[SORT_BLOCK], sval[SORT_BLOCK];
    __shared__ float sscale[SORT_BLOCK];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, first = w * (64 * PASS_ITEMS) + lane;
    const long block = (long)blockIdx.x * SORT_BLOCK;
    const int n = (int)(a.n - block < SORT_BLOCK ? a.n - block : SORT_BLOCK);
    const uint32_t mask = (1u << p.bits) - 1u;
    const unsigned long long before = (1ull << lane) - 1ull;
    for (int d = threadIdx.x; d < PASS_WAVES * 256; d += PASS_THREADS) (&cnt[0][0])[d] = 0;
    uint32_t key[PASS_ITEMS], val[PASS_ITEMS], rank[PASS_ITEMS];
    float scale[PASS_ITEMS];
#pragma unroll
    for (int x = 0; x < PASS_ITEMS; ++x) {
        const int i = first + 64 * x;
        const bool in = i < n;
        key[x] = in ? pass_key(a, p, block + i) : NO_ENTRY;
        val[x] = in && p.val ? p.val[block + i] : (uint32_t)(block + i);
        scale[x] = in && p.scale ? p.scale[block + i] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < PASS_ITEMS; ++x) {
        const bool in = first + 64 * x < n;
        const uint32_t d = (key[x] >> p.shift) & mask;
        unsigned long long same = __ballot(in);
        for (int b = 0; b < p.bits; ++b) {
            const unsigned long long on = __ballot((d >> b) & 1u);
            same &= ((d >> b) & 1u) ? on : ~on;
        }
        const uint32_t prior = cnt[w][d];
        rank[x] = prior + (uint32_t)__popcll(same & before);
        wave_order();
        if (in && (same & before) == 0) cnt[w][d] = prior + (uint32_t)__popcll(same);
        wave_order();
    }
    __syncthreads();
    // per digit: where the waves' entries begin in the block, and where the block's begin among all
    uint32_t total = 0, incl = 0, all = 0, all_incl = 0;
    if (threadIdx.x < 256) {
        for (int k = 0; k < PASS_WAVES; ++k) {
            const uint32_t c = cnt[k][threadIdx.x];
            cnt[k][threadIdx.x] = total;
            total += c;
        }
        all = threadIdx.x <= mask ? p.totals[threadIdx.x] : 0u;
        incl = total;
        all_incl = all;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)incl, d, 64), q = (uint32_t)__shfl_up((int)all_incl, d, 64);
            if (lane >= d) { incl += o; all_incl += q; }
        }
        if (lane == 63) { wave_sum[0][w] = incl; wave_sum[1][w] = all_incl; }
    }
    __syncthreads();
    if (threadIdx.x < 256) {
        uint32_t l = incl - total, g = all_incl - all;
        for (int k = 0; k < w; ++k) { l += wave_sum[0][k]; g += wave_sum[1][k]; }
        local[threadIdx.x] = l;
        global[threadIdx.x] = threadIdx.x <= mask ? g + p.hist[(size_t)threadIdx.x * p.blocks + blockIdx.x] : 0u;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < PASS_ITEMS; ++x) {
        if (first + 64 * x < n) {
            const uint32_t d = (key[x] >> p.shift) & mask, at = local[d] + cnt[w][d] + rank[x];
            skey[at] = key[x];
            sval[at] = val[x];
            sscale[at] = scale[x];
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += PASS_THREADS) {
        const uint32_t k = skey[j], d = (k >> p.shift) & mask, to = global[d] + ((uint32_t)j - local[d]);
        p.key_out[to] = k;
        p.val_out[to] = sval[j];
        if (p.scale) p.scale_out[to] = sscale[j];
    }
}

// ---- the sums of the table's gradient over the sorted entries.
//
// Split by ENTRIES, not by rows, so that a row hit a million times costs what a million rows hit once do: a group of G lanes
// (V columns each; G x V covers the width, or a tile of it) takes a chunk of consecutive sorted entries, keeps the running sum of the
// current row in registers and stores it where the row changes.  A row that begins and ends inside the chunk goes straight to the
// gradient; the sum of one that crosses the chunk's border goes to a slot of its own -- head: of the row that came in from the chunk
// before; tail: of the row that begins here and goes on -- and k_lookup_join adds a row's tail and the heads behind it in order.
// No atomics, and every order fixed by the sizes and the ids.
//
// The gradient rows are gathered: each is one contiguous read of width x 4 bytes, UNROLL of them in flight per lane.  ONCE: streamed,
// where the gradient is larger than the 256 MB cache in front of the memory.  (Rows of 45 floats, right after the kernel that wrote them:
// 54 MB 44 us streamed and 30 as other reads, 108 MB 53 and 33, 180 MB 76 and 66, 360 MB 144 and 149.)
constexpr int UNROLL = 8;
constexpr long SUM_ONCE_BYTES = 256l << 20;

struct SumArgs {
    const uint32_t *key, *val;
    const float* scales;          // in the entries' sorted order; NULL: row_scale by entry
    const void* grad;
    long grad_stride;
    void* d_table;
    float* d_row_scale;
    float* slots;                 // [chunks][2][width]: head, tail
    int chunk;                    // entries of a chunk, a multiple of UNROLL
    int g_shift;                  // G = 1 << g_shift lanes
};

template <typename TT, typename TO, int V, bool DSCALE, bool ONCE>
__global__ void __launch_bounds__(256) k_lookup_sum(LookupArgs a, SumArgs q)
{
    constexpr int U = UNROLL, U_SHIFT = 3;
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
    uint32_t cur = q.key[first];
    bool came_in = first > 0 && q.key[first - 1] == cur;
    Pack<TT, V> t_cur;
    if (DSCALE && cur < rows) t_cur = *reinterpret_cast<const Pack<TT, V>*>(table + (long)cur * a.table_stride);
    float acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.0f;
    for (long j = first; j < last; j += U) {
        // (the arrays are padded to whole chunks: the loads need no bounds, what lies behind `last` is masked)
        uint4 k4[U / 4], v4[U / 4];
#pragma unroll
        for (int x = 0; x < U / 4; ++x) {
            k4[x] = reinterpret_cast<const uint4*>(q.key + j)[x];
            v4[x] = reinterpret_cast<const uint4*>(q.val + j)[x];
        }
        uint32_t key[U], val[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const bool in = j + x < last;
            key[x] = in ? (&k4[x / 4].x)[x % 4] : NO_ENTRY;
            val[x] = in ? (&v4[x / 4].x)[x % 4] : 0u;
        }
        Pack<TO, V> g[U];
        float s[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            const bool there = key[x] < rows;
            s[x] = q.scales ? q.scales[j + x] : there && a.row_scale ? a.row_scale[val[x]] : 1.0f;     // (padded as the keys)
            g[x] = load_pack<TO, V, ONCE>(grad + (there ? (long)val[x] * q.grad_stride : 0));
        }
        float dot[U];
#pragma unroll
        for (int x = 0; x < U; ++x) {
            if (key[x] != cur && key[x] != NO_ENTRY) {
                if (live && cur < rows) {
                    if (came_in) store_row<float, V>(slot, acc);
                    else store_row<TT, V>(d_table + (long)cur * a.width, acc);
                }
                came_in = false;
                cur = key[x];
                // (the row of the table is waited for here: reading all that begin among the U ahead of time takes registers for
                // eight of them and with those a wave per SIMD -- 152 us against 141 at 244 entries a row, 192 against 195 at 4,
                // 282 against 297 at one)
                if (DSCALE && cur < rows) t_cur = *reinterpret_cast<const Pack<TT, V>*>(table + (long)cur * a.table_stride);
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
                    if (DSCALE && col + v >= want) dot[x] = fmaf(gv, load_f32(t_cur.v + v), dot[x]);
                }
                if (DSCALE) dot[x] *= a.scale;
            }
        }
        if (DSCALE) {
            // the group's sums of the U products.  Where it has as many lanes, half of them pass on the half of the sums
            // that the others keep, three times, so that every eighth of the lanes ends with one sum: 8 exchanges and one store
            // for 16 lanes where a butterfly for each sum takes 32 and eight (2 M x 45: 3 % of the kernel)
            float d[U];
#pragma unroll
            for (int x = 0; x < U; ++x) d[x] = live ? dot[x] : 0.0f;
            if (q.g_shift >= U_SHIFT) {
                int w = G >> 1;
#pragma unroll
                for (int half = U / 2; half > 0; half >>= 1, w >>= 1) {
                    const bool high = (lane & w) != 0;
#pragma unroll
                    for (int x = 0; x < half; ++x) {
                        const float keep = high ? d[x + half] : d[x], pass = high ? d[x] : d[x + half];
                        d[x] = keep + __shfl_xor(pass, w, 64);
                    }
                }
                for (; w > 0; w >>= 1) d[0] += __shfl_xor(d[0], w, 64);
                const int x = lane >> (q.g_shift - U_SHIFT);
                if ((lane & ((G >> U_SHIFT) - 1)) == 0 && j + x < last) q.d_row_scale[q.val[j + x]] = d[0];
            } else {
#pragma unroll
                for (int x = 0; x < U; ++x) {
                    for (int w = G >> 1; w > 0; w >>= 1) d[x] += __shfl_xor(d[x], w, 64);
                    if (lane == 0 && j + x < last) q.d_row_scale[val[x]] = d[x];
                }
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

// Rows that cross borders of chunks: tail[c] + head[c + 1] + ... + head[end].  A workgroup looks at up to JOIN_CHUNKS chunks; short
// rows are one group's each, rows of more than JOIN_LONG pieces the whole workgroup's: group k adds the pieces k, k + groups, ... and
// the groups' sums are added pairwise.  A group adds at most JOIN_RUN pieces in a row, then at most JOIN_RUN such sums, then those: with
// the 64 entries of a chunk and the 10 steps between 1024 groups at most 394 additions lie between an entry and the result, for the
// 2^20 pieces a group that 2^30 entries of one row make as well.  (One running sum: 511 u off after 2^21 equal entries, 35 u like this.)
constexpr int JOIN_THREADS = 1024, JOIN_CHUNKS = 64, JOIN_LONG = 16, JOIN_AHEAD = 8, JOIN_RUN = 128;

// The sums of a workgroup's groups, pairwise: group 0's lanes hold the result.  part: V floats for every thread, free before.
template <int V>
__device__ __forceinline__ void add_groups(float (&acc)[V], float* part, int g_shift)
{
    const int group = threadIdx.x >> g_shift;
#pragma unroll
    for (int v = 0; v < V; ++v) part[threadIdx.x * V + v] = acc[v];
    __syncthreads();
    for (int w = (int)(blockDim.x >> g_shift) >> 1; w > 0; w >>= 1) {
        if (group < w) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                acc[v] += part[(threadIdx.x + (w << g_shift)) * V + v];
                part[threadIdx.x * V + v] = acc[v];
            }
        }
        __syncthreads();
    }
}

// acc += the pieces p, p + step, ... up to `end` of the row whose tail is piece c, JOIN_AHEAD of them in flight.  RUNS: any number of
// them, in runs of JOIN_RUN.
template <int V, bool RUNS>
__device__ __forceinline__ void join_pieces(float (&acc)[V], const float* __restrict__ slots, long width, long c, long p, long end,
                                            long step)
{
    float runs[V], sums[V];
    int in_run = JOIN_RUN / JOIN_AHEAD, in_runs = JOIN_RUN;
#pragma unroll
    for (int v = 0; v < V; ++v) runs[v] = sums[v] = 0.0f;
#pragma unroll 1
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
        if (RUNS && --in_run == 0) {
            in_run = JOIN_RUN / JOIN_AHEAD;
#pragma unroll
            for (int v = 0; v < V; ++v) { runs[v] += acc[v]; acc[v] = 0.0f; }
            if (--in_runs == 0) {
                in_runs = JOIN_RUN;
#pragma unroll
                for (int v = 0; v < V; ++v) { sums[v] += runs[v]; runs[v] = 0.0f; }
            }
        }
    }
    if (RUNS) {
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = sums[v] + (runs[v] + acc[v]);
    }
}

// (V == 4: registers for two workgroups on a CU, which the compiler does not keep to by itself)
template <typename TT, int V>
__global__ void __launch_bounds__(JOIN_THREADS, V == 4 ? 8 : 4) k_lookup_join(LookupArgs a, SumArgs q, long chunks, int each)
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
        const long c = (long)blockIdx.x * each + threadIdx.x, first = c * q.chunk, next = first + q.chunk;
        bool owner = false;
        uint32_t k = 0;
        if ((int)threadIdx.x < each && c < chunks && next < a.n) {
            k = q.key[next - 1];
            // its last row goes on, and begins in this chunk
            owner = k < (uint32_t)a.rows && q.key[next] == k && (first == 0 || q.key[first - 1] != k);
        }
        const unsigned long long mask = __ballot(owner);           // (one wave: JOIN_CHUNKS is 64)
        if (threadIdx.x == 0) count = __popcll(mask);
        if (owner) {
            const int at = __popcll(mask & ((1ull << threadIdx.x) - 1ull));
            from[at] = c; row[at] = k;
            // the last chunk whose first entry is of the row: one of the next four, or (-1) further on
            int more = 0;
            bool on = true;
#pragma unroll
            for (int x = 1; x <= 4; ++x) {
                const long p = c + 1 + x < chunks ? c + 1 + x : c;
                const bool same = q.key[p * q.chunk] == k && p != c;
                on = on && same;
                more += on;
            }
            upto[at] = more < 4 ? c + 1 + more : -1;
        }
    }
    __syncthreads();
    // longer rows, a wave per row: chunks 1, 2, 4, ... further on at once, then 64 in between
    for (int o = threadIdx.x >> 6; o < count; o += JOIN_THREADS / 64) {
        if (upto[o] >= 0) continue;
        const long base = from[o] + 1;
        const uint32_t k = row[o];
        const int at = threadIdx.x & 63;
        long lo = 0, x = at < 31 ? 1l << at : chunks;
        unsigned long long off = ~__ballot(base + x < chunks && q.key[(base + (base + x < chunks ? x : 0)) * q.chunk] == k);
        const int t = __ffsll(off) - 1;                            // (lane 63 is always off)
        lo = t == 0 ? 0 : 1l << (t - 1);
        long hi = 1l << t;                                         // not of the row, or behind the last chunk
        if (hi > chunks - base) hi = chunks - base;
        while (hi - lo > 1) {
            const long step = (hi - lo + 63) / 64;
            x = lo + (at + 1) * step;
            off = ~__ballot(x < hi && q.key[(base + (x < hi ? x : lo)) * q.chunk] == k);
            const int more = off == 0 ? 64 : __ffsll(off) - 1;
            lo += more * step;
            if (lo + step < hi) hi = lo + step;
        }
        if (at == 0) upto[o] = base + lo;
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
        join_pieces<V, false>(acc, slots, a.width, c, c, end, 1);
        store_row<TT, V>(d_table + (long)row[o] * a.width, acc);
    }
    for (int o = 0; o < count; ++o) {
        const long c = from[o], end = upto[o];
        if (end - c <= JOIN_LONG) continue;                         // (the same for every thread)
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.0f;
        join_pieces<V, true>(acc, slots, a.width, c, c + group, end, groups);
        __syncthreads();
        add_groups<V>(acc, part, q.g_shift);
        if (group == 0 && live) store_row<TT, V>(d_table + (long)row[o] * a.width, acc);
    }
}

// ---- up to SMALL entries in one launch without any scratch: every workgroup sorts all of them in its LDS and writes the rows of its own
// range, the ones without entries as zeros.  A row is one group's; one of more than SMALL_LONG entries is the whole workgroup's, in
// contiguous pieces that are added pairwise.  (100 entries, 1000 rows of ten floats: 9 us against 12 in three launches.)
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
            g[x] = load_pack<TO, V, false>(grad + i * q.grad_stride);
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
    const int n = (int)a.n;
    if (threadIdx.x == 0) n_long = 0;
    if ((int)threadIdx.x < n) {
        lds.key[threadIdx.x] = key_of(a, threadIdx.x);
        lds.val[threadIdx.x] = threadIdx.x;
    }
    __syncthreads();
    sort_in_lds<1>(lds, n, 0, bits);
    const int G = 1 << q.g_shift, lane = threadIdx.x & (G - 1), group = threadIdx.x >> q.g_shift, groups = SORT_THREADS >> q.g_shift;
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
        add_groups<V>(acc, part, q.g_shift);
        if (group == 0 && live) store_row<TT, V>(d_table + (long)k * a.width, acc);
        __syncthreads();
    }
}

// The scales' gradient alone, entry by entry: where the table's is not wanted, or the width takes more than one tile.
template <typename TT, typename TO, int V>
__global__ void __launch_bounds__(256) k_lookup_dscale(LookupArgs a, const TO* __restrict__ grad, long grad_stride,
                                                       float* __restrict__ d_row_scale, int g_shift)
{
    const int G = 1 << g_shift, lane = threadIdx.x & (G - 1);
    const long i = (((long)blockIdx.z * gridDim.x + blockIdx.x) * 256 + threadIdx.x) >> g_shift;
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
    if (lane == 0) d_row_scale[i] = row >= 0 ? a.scale * acc : 0.0f;
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
    // long chunks make few slots; shorter ones while there are fewer than four waves for each of the 1024 SIMDs (16384 entries of 1024
    // 16-bit values: 13 us with four, 19 with one) -- but not so short that a row that all entries hit has more than JOIN_RUN pieces
    // for each group of a join, which takes them one after the other (at 64 entries, of more than 8192 a group, it has)
    t.chunk = 64;
    const int64_t most = JOIN_RUN * (JOIN_THREADS >> t.g_shift);
    while (t.chunk > UNROLL && ((n << t.g_shift) / 64 / t.chunk) * t.tiles < 4096 && 2 * n <= most * t.chunk) t.chunk >>= 1;
    t.chunks = (long)((n + t.chunk - 1) / t.chunk);
    return t;
}

// A grid of `blocks` workgroups by `tiles`.  A launch has fewer than 2^32 threads in x, which 2^24 workgroups of 256 would be:
// more than 2^20 go on in z.
static dim3 grid_of(int64_t blocks, int tiles)
{
    const int64_t x = blocks < 1 ? 1 : blocks < (1 << 20) ? blocks : 1 << 20;
    return dim3((unsigned)x, (unsigned)tiles, (unsigned)((blocks + x - 1) / x));
}

static int check_lookup(const VrLookup* l, LookupArgs& a)
{
    if (!l) { set_error("lookup: arguments are required"); return VR_ERR_INVALID_ARGUMENT; }
    if (l->n < 0 || l->n >= (1ll << 30) || l->rows < 0 || l->rows >= 0x7fffffffll || l->width < 1 || l->width > (1 << 22) ||
        l->table_stride < l->width || l->table_stride > (1ll << 40))
        { set_error("lookup: need 0 <= n < 2^30, 0 <= rows < 2^31 - 1, 1 <= width <= 2^22, table_stride >= width"); return VR_ERR_INVALID_ARGUMENT; }
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
        const dim3 grid = grid_of((a.n + per - 1) / per, t.tiles);
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
    template <typename TT, typename TO, int V, bool ONCE>
    static void sums(const LookupArgs& a, const SumArgs& q, const Tiling& t, bool fused, hipStream_t s)
    {
        const dim3 grid((unsigned)(((t.chunks << t.g_shift) + 255) / 256), t.tiles);
        if (fused) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_sum<TT, TO, V, true, ONCE>), grid, dim3(256), 0, s, a, q);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_sum<TT, TO, V, false, ONCE>), grid, dim3(256), 0, s, a, q);
    }
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
            if (V > 1 && a.n * a.width * (long)sizeof(TO) > SUM_ONCE_BYTES) sums<TT, TO, V, V != 1>(a, q, t, fused, s);
            else sums<TT, TO, V, false>(a, q, t, fused, s);
            // (few chunks: fewer a workgroup, so that each of its groups has one row at most.  8125 chunks of 45 floats: 5 us with 16, 8
            // with 64; 31250: 19 and 13)
            const int each = t.chunks > 8192 ? JOIN_CHUNKS : JOIN_CHUNKS / 4;
            if (t.chunks > 1)
                hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_join<TT, V>), dim3((unsigned)((t.chunks + each - 1) / each), t.tiles),
                                   dim3(JOIN_THREADS), 0, s, a, q, t.chunks, each);
        }
        if (q.d_row_scale && !fused)
            hipLaunchKernelGGL(HIP_KERNEL_NAME(k_lookup_dscale<TT, TO, V>), grid_of(((a.n << t.g_shift) + 255) / 256, 1), dim3(256),
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

// scratch: two sets of keys, values and scales, the sort's counts, and the slots of the chunks
struct Scratch {
    size_t array, arrays, hist, slots;      // bytes of one array, of all, of the counts and totals, of the slots
    int blocks;
};
static Scratch scratch_of(int64_t n, int64_t width)
{
    Scratch s;
    s.array = align_up((size_t)n * 4, 256);         // (whole chunks of 64 entries)
    s.blocks = (int)((n + SORT_BLOCK - 1) / SORT_BLOCK);
    s.arrays = n <= SORT_SMALL ? 2 * s.array : 6 * s.array;
    s.hist = n <= SORT_SMALL ? 0 : align_up(256 * (size_t)s.blocks * 4 + 256 * 4, 256);
    const long chunks = tiling(n, width, 4).chunks > tiling(n, width, 8).chunks ? tiling(n, width, 4).chunks : tiling(n, width, 8).chunks;
    s.slots = align_up((size_t)chunks * 2 * (size_t)width * sizeof(float), 256);
    return s;
}

extern "C" int64_t vr_lookup_scratch_bytes(int64_t n, int64_t rows, int64_t width)
{
    if (n < 0 || n >= (1ll << 30) || rows < 0 || rows >= 0x7fffffffll || width < 1 || width > (1 << 22)) return 0;
    if (n <= SMALL) return 0;
    const Scratch s = scratch_of(n, width);
    return (int64_t)(s.arrays + s.hist + s.slots);
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
    if (a.n == 0) d_row_scale = nullptr;                // (without entries there is only the table's gradient to clear)
    if (!d_table && !d_row_scale) return VR_OK;
    hipStream_t s = (hipStream_t)stream;
    SumArgs q{nullptr, nullptr, nullptr, grad, (long)grad_stride, d_table, d_row_scale, nullptr, 0, 0};
    if (d_table && a.n > SMALL) {
        const Scratch sc = scratch_of(a.n, a.width);
        char* base = (char*)scratch;
        uint32_t *key[2], *val[2];
        float* scale[2];
        for (int k = 0; k < 2; ++k) {
            key[k] = (uint32_t*)(base + (a.n <= SORT_SMALL ? 0 : k) * 3 * sc.array);
            val[k] = key[k] + sc.array / 4;
            scale[k] = (float*)(val[k] + sc.array / 4);
        }
        q.slots = (float*)(base + sc.arrays + sc.hist);
        const long zero_bytes = a.rows * a.width * (long)t_element, zero_blocks = (zero_bytes + 16383) / 16384;
        const int bits = key_bits(a.rows);
        if (a.n <= SORT_SMALL) {
            const dim3 grid(SORT_GROUPS + (unsigned)(zero_blocks < 1024 ? zero_blocks : 1024));
            const uint32_t range = (uint32_t)((a.rows + SORT_GROUPS) / SORT_GROUPS);          // of the keys 0 .. rows
            hipLaunchKernelGGL(k_lookup_sort, grid, dim3(SORT_THREADS), 0, s, a, key[0], val[0], range, key_bits((int64_t)range - 1),
                               (char*)d_table, zero_bytes);
            VR_KERNEL_CHECK("lookup_sort", s, false);
            q.key = key[0];
            q.val = val[0];
        } else {
            const int passes = (bits + 7) / 8;
            PassArgs p{nullptr, nullptr, a.row_scale, nullptr, nullptr, nullptr, (uint32_t*)(base + sc.arrays), nullptr, sc.blocks, 0, 0};
            p.totals = p.hist + 256 * (size_t)sc.blocks;
            for (int pass = 0, to = 0; pass < passes; ++pass, to ^= 1) {
                p.bits = (bits - p.shift + passes - pass - 1) / (passes - pass);          // as even as they get
                p.key_out = key[to]; p.val_out = val[to]; p.scale_out = scale[to];
                const unsigned zeros = pass > 0 ? 0 : (unsigned)(zero_blocks < 2048 ? zero_blocks : 2048);
                hipLaunchKernelGGL(k_sort_hist, dim3(sc.blocks + zeros), dim3(PASS_THREADS), 0, s, a, p, (char*)d_table, zero_bytes);
                hipLaunchKernelGGL(k_sort_sums, dim3(1u << p.bits), dim3(256), 0, s, p);
                hipLaunchKernelGGL(k_sort_scatter, dim3(sc.blocks), dim3(PASS_THREADS), 0, s, a, p);
                VR_KERNEL_CHECK("lookup_sort", s, false);
                p.key = p.key_out; p.val = p.val_out;
                if (p.scale) p.scale = p.scale_out;
                p.shift += p.bits;
            }
            q.key = p.key;
            q.val = p.val;
            q.scales = p.scale;
        }
    }
    return by_type<Backward>(lookup, a, q, s);
}
