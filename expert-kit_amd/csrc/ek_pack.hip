// Routing / pack kernels: (token, slot) -> per-expert contiguous segments.
//
// Reproduces, as a stable counting sort, the grouping that
// NaiveExecutor::break_down_to_egress builds with per-expert push lists
// (ek-computation/src/controller/executor.rs:283-304): within an expert's
// segment the pairs keep ascending flat index t*K + k.
//
// Three launches, all integer work, all HBM/LDS bound:
//   pack_hist : one LDS histogram per 4096-pair chunk
//   pack_scan : per-expert exclusive scan over chunks, then a wavefront
//               prefix scan over experts -> counts, offsets, and the FFN
//               kernels' work lists
//   pack_rank : stable rank of every pair inside its chunk by wave-level
//               match (ballots over the id bits) -> perm, inv_perm, row_token
// (calls of at most 4096 pairs run all of it in one workgroup, pack_fused)
// plus a coalesced row gather (assemble_seq_tensors, executor.rs:112-133).
#include "ek_internal.h"
#include "ek_quant.h"

namespace ek {

__global__ __launch_bounds__(kPackThreads) void pack_hist_kernel(PackArgs a)
{
    __shared__ int32_t hist[kMaxExperts];
    for (int i = threadIdx.x; i < a.E; i += kPackThreads) hist[i] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * kPackChunk;
    const int64_t end = min(base + (int64_t)kPackChunk, a.P);
    // (ids out of range are left out; the scan kernel sees that the counts do not add up to P)
    int32_t id[kPackChunk / kPackThreads];                // all loads in flight at once
#pragma unroll
    for (int u = 0; u < kPackChunk / kPackThreads; ++u) {
        const int64_t p = base + u * kPackThreads + threadIdx.x;
        id[u] = p < end ? a.ids[p] : -1;
    }
#pragma unroll
    for (int u = 0; u < kPackChunk / kPackThreads; ++u)
        if ((uint32_t)id[u] < (uint32_t)a.E) atomicAdd(&hist[id[u]], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < a.E; i += kPackThreads)
        a.block_hist[(int64_t)blockIdx.x * a.E + i] = hist[i];
}

// Exclusive prefix sums of five ints per thread over a 1024-thread workgroup (the offsets and the four
// work lists' positions), with one pair of barriers: shuffles inside each wavefront, then the 16 wave
// totals through LDS.  wave_tot: [16][5].
__device__ __forceinline__ void block_exclusive_scan5(const int32_t (&v)[5], int32_t (*wave_tot)[5],
                                                      int32_t (&excl)[5], int32_t (&total)[5])
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t incl[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) incl[i] = v[i];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            const int32_t up = __shfl_up(incl[i], d, 64);
            if (lane >= d) incl[i] += up;
        }
    }
    __syncthreads();   // wave_tot may still be read from a previous scan
    if (lane == 63) {
#pragma unroll
        for (int i = 0; i < 5; ++i) wave_tot[wave][i] = incl[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 5; ++i) {
        int32_t base = 0, sum = 0;
        for (int w = 0; w < 16; ++w) {
            const int32_t t = wave_tot[w][i];
            if (w < wave) base += t;
            sum += t;
        }
        asm volatile("" : "+v"(base), "+v"(sum));  // sums of this place: the sixteen totals need not live until their use
        total[i] = sum;
        excl[i] = base + incl[i] - v[i];
    }
}

// How one segment of n rows is cut into work items (see WorkLists).
struct SegmentCut {
    int32_t n128, n64, n32, ns;
};
__device__ __forceinline__ SegmentCut cut_segment(int32_t n, int32_t one_class)
{
    SegmentCut c;
    if (one_class) {
        if (one_class == 3) {
            c.n128 = c.n64 = c.n32 = 0;
            c.ns = (n + kWideRows - 1) / kWideRows;
            return c;
        }
        const bool tile = one_class == 2 ? n > 0 : n > 16;
        c.n128 = tile ? q8_items(n) : 0;
        c.n64 = c.n32 = 0;
        c.ns = n > 0 && !tile;
        return c;
    }
    const int32_t r = n & 127;
    c.n128 = (n >> 7) + (r > 64);
    c.n64 = r > 32 && r <= 64;
    c.n32 = r > 16 && r <= 32;
    c.ns = r > 0 && r <= 16;
    return c;
}
__device__ __forceinline__ bool in_one_class(const WorkLists &l, int32_t n) { return l.one_class == 2 ? n > 0 : l.one_class == 1 && n > 16; }
__device__ __forceinline__ WorkItem q8_work_item(int32_t e, int32_t seg0, int32_t n, int32_t items, int32_t i)
{
    int32_t first, rows;
    q8_item(n, items, i, &first, &rows);
    return WorkItem{e, seg0 + first, rows, 0};
}
// The items of a segment of n rows from seg0 on, at their positions in the lists: as many of each class as
// cut_segment says.  The callers' `threads` threads (this one is number `tid`) share the work.
__device__ __forceinline__ void emit_items(const WorkLists &l, int32_t e, int32_t seg0, int32_t n, int32_t p128, int32_t p64,
                                           int32_t p32, int32_t ps, int32_t tid = 0, int32_t threads = 1)
{
    if (l.one_class == 3) {
        for (int32_t i = tid; i * kWideRows < n; i += threads)
            l.items[kListStream][ps + i] = WorkItem{e, seg0 + i * kWideRows, min(kWideRows, n - i * kWideRows), 0};
        return;
    }
    if (in_one_class(l, n)) {
        const int32_t items = q8_items(n);
        for (int32_t i = tid; i < items; i += threads) l.items[kListT128][p128 + i] = q8_work_item(e, seg0, n, items, i);
        return;
    }
    const int32_t full = n >> 7, r = n & 127;
    for (int32_t t = tid; t < full; t += threads) l.items[kListT128][p128 + t] = WorkItem{e, seg0 + t * 128, 128, 0};
    if (tid != 0) return;
    const WorkItem rem{e, seg0 + full * 128, r, 0};
    if (r > 64) l.items[kListT128][p128 + full] = rem;
    else if (r > 32) l.items[kListT64][p64] = rem;
    else if (r > 16) l.items[kListT32][p32] = rem;
    else if (r > 0) l.items[kListStream][ps] = rem;
}

// One workgroup of 1024 threads; thread e owns expert e.
__global__ __launch_bounds__(1024) void pack_scan_kernel(PackArgs a)
{
    __shared__ int32_t wave_tot[16][5];
    const int e = threadIdx.x;
    int32_t total = 0;
    const bool absent = e < a.E && a.slabs != nullptr && a.slabs[e].upgate == nullptr;
    if (e < a.E) {
        // exclusive prefix over chunks, 16 chunks' counts in flight at a time (one dependent load
        // per chunk made this kernel's time: 10 us at 9 chunks)
        for (int b0 = 0; b0 < a.nblocks; b0 += 16) {
            int32_t v[16];
#pragma unroll
            for (int u = 0; u < 16; ++u)
                v[u] = b0 + u < a.nblocks ? a.block_hist[(int64_t)(b0 + u) * a.E + e] : 0;
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                if (b0 + u < a.nblocks) a.block_hist[(int64_t)(b0 + u) * a.E + e] = total;
                total += v[u];
            }
        }
        a.counts[e] = total;
        if (a.activation) a.activation[e] += (uint64_t)total;
    }
    const int any_unloaded = __syncthreads_or(absent && total > 0);
    const SegmentCut c = cut_segment(total, a.lists.one_class);
    const int32_t v5[5] = {total, c.n128, c.n64, c.n32, c.ns};
    int32_t ex[5], tot5[5];
    block_exclusive_scan5(v5, wave_tot, ex, tot5);
    const int32_t off = ex[0], sum = tot5[0];
    if (e < a.E) a.offsets[e] = off;
    if (e == 0) {
        a.offsets[a.E] = sum;
        // the error word is written, not accumulated: every pair with an id in range was counted once
        a.err[0] = ((int64_t)sum != a.P ? 1 : 0) | (any_unloaded ? 2 : 0);
    }
    if (a.lists.count == nullptr) return;
    if (e < a.E && total > 0) emit_items(a.lists, e, off, total, ex[1], ex[2], ex[3], ex[4]);
    if (e == 0) {
        a.lists.count[kListT128] = tot5[1];
        a.lists.count[kListT64] = tot5[2];
        a.lists.count[kListT32] = tot5[3];
        a.lists.count[kListStream] = tot5[4];
        if (a.tile_items_host) *a.tile_items_host = tot5[1] + tot5[2] + tot5[3];
    }
}

// Work lists that hold one segment and nothing else: rows row0 .. row0+n-1 of expert e.
// mode 0: the usual cut; 1: 16-row streaming items; 2: streaming items of up to kWideRows rows.
// row_token, if given, maps the segment's rows to tokens 0 .. n-1.
__global__ __launch_bounds__(256) void segment_lists_kernel(WorkLists l, int32_t e, int32_t row0, int32_t n,
                                                            int32_t *row_token, int32_t mode)
{
    if (row_token)
        for (int32_t t = threadIdx.x; t < n; t += 256) row_token[row0 + t] = t;
    if (mode) {
        const int32_t per = mode == 2 ? kWideRows : 16, items = (n + per - 1) / per;
        for (int32_t t = threadIdx.x; t < items; t += 256)
            l.items[kListStream][t] = WorkItem{e, row0 + t * per, min(per, n - t * per), 0};
        if (threadIdx.x == 0) {
            l.count[kListT128] = l.count[kListT64] = l.count[kListT32] = 0;
            l.count[kListStream] = items;
        }
        return;
    }
    const SegmentCut c = cut_segment(n, l.one_class);
    emit_items(l, e, row0, n, 0, 0, 0, 0, threadIdx.x, 256);
    if (threadIdx.x == 0) {
        l.count[kListT128] = c.n128;
        l.count[kListT64] = c.n64;
        l.count[kListT32] = c.n32;
        l.count[kListStream] = c.ns;
    }
}

__global__ __launch_bounds__(256) void append_segment_kernel(WorkLists l, int32_t e, int32_t row0, int32_t n,
                                                             int32_t *row_token, int32_t as_stream)
{
    const int32_t p128 = l.count[kListT128], p64 = l.count[kListT64], p32 = l.count[kListT32],
                  ps = l.count[kListStream];
    __syncthreads();   // every thread has read the old lengths before thread 0 replaces them
    if (as_stream) {
        // a decode-sized segment: as one tile per 128 rows it would run on a handful of CUs for
        // the length of the whole contraction; as streaming items it spreads over the chip.
        // as_stream = 1: 16-row items appended to the list; 2: items of up to kWideRows rows
        // that become the whole list (a list of their own, for a launch of their own)
        const int32_t per = as_stream == 2 ? kWideRows : 16, at = as_stream == 2 ? 0 : ps;
        const int32_t items = (n + per - 1) / per;
        for (int32_t t = threadIdx.x; t < items; t += 256)
            l.items[kListStream][at + t] = WorkItem{e, row0 + t * per, min(per, n - t * per), 0};
        for (int32_t t = threadIdx.x; t < n; t += 256) row_token[row0 + t] = t;
        if (threadIdx.x == 0) l.count[kListStream] = at + items;
        return;
    }
    const SegmentCut c = cut_segment(n, l.one_class);
    for (int32_t t = threadIdx.x; t < n; t += 256) row_token[row0 + t] = t;
    emit_items(l, e, row0, n, p128, p64, p32, ps, threadIdx.x, 256);
    if (threadIdx.x == 0) {
        l.count[kListT128] = p128 + c.n128;
        l.count[kListT64] = p64 + c.n64;
        l.count[kListT32] = p32 + c.n32;
        l.count[kListStream] = ps + c.ns;
    }
}

void launch_append_segment(const WorkLists &lists, int32_t expert, int32_t row0, int32_t n, int32_t *row_token,
                           int as_stream, hipStream_t s)
{
    hipLaunchKernelGGL(append_segment_kernel, dim3(1), dim3(256), 0, s, lists, expert, row0, n, row_token,
                       as_stream);
}

void launch_single_lists(const WorkLists &lists, int32_t expert, int32_t n, bool wide, hipStream_t s)
{
    hipLaunchKernelGGL(segment_lists_kernel, dim3(1), dim3(256), 0, s, lists, expert, 0, n, (int32_t *)nullptr, wide ? 2 : 0);
}

void launch_segment_lists(const WorkLists &lists, int32_t expert, int32_t row0, int32_t n, int32_t *row_token, int mode,
                          hipStream_t s)
{
    hipLaunchKernelGGL(segment_lists_kernel, dim3(1), dim3(256), 0, s, lists, expert, row0, n, row_token, mode);
}

// 16 waves per chunk of 4096 pairs: a wave's 256 pairs are four dependent steps on its counters (65536 pairs on MI355X:
// 10 us, 20 with four waves that load the ids again at every step).
constexpr int kRankThreads = 1024;
__global__ __launch_bounds__(kRankThreads) void pack_rank_kernel(PackArgs a, int nbits)
{
    constexpr int kWaves = kRankThreads / 64;
    constexpr int kSub = kPackChunk / kWaves;   // pairs per wave, consecutive
    extern __shared__ int32_t rank_lds[];                 // wbase[kWaves][E]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t *wbase = rank_lds + wave * a.E;
    const int64_t start = (int64_t)blockIdx.x * kPackChunk + (int64_t)wave * kSub;
    // the wave's ids, loaded once: one memory latency instead of one per 64 pairs in either loop below
    int32_t ids[kSub / 64];
#pragma unroll
    for (int it = 0; it < kSub / 64; ++it) {
        const int64_t p = start + it * 64 + lane;
        ids[it] = p < a.P ? a.ids[p] : -1;
    }
    for (int i = threadIdx.x; i < kWaves * a.E; i += kRankThreads) rank_lds[i] = 0;
    __syncthreads();
#pragma unroll
    for (int it = 0; it < kSub / 64; ++it)
        if ((uint32_t)ids[it] < (uint32_t)a.E) atomicAdd(&wbase[ids[it]], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kRankThreads) {
        int32_t run = a.offsets[e] + a.block_hist[(int64_t)blockIdx.x * a.E + e];
        for (int w = 0; w < kWaves; ++w) {
            const int32_t t = rank_lds[w * a.E + e];
            rank_lds[w * a.E + e] = run;
            run += t;
        }
    }
    __syncthreads();
    // Each wave walks its own consecutive pairs 64 at a time; lanes holding
    // the same expert id find each other with one ballot per id bit, so the
    // rank inside the group is the number of lower lanes in the group.
#pragma unroll
    for (int it = 0; it < kSub / 64; ++it) {
        const int64_t p = start + it * 64 + lane;
        const int32_t id = ids[it];
        const bool valid = (uint32_t)id < (uint32_t)a.E;
        if (!valid && p < a.P) a.inv_perm[p] = -1;
        uint64_t m = __ballot(valid);
        for (int b = 0; b < nbits; ++b) {
            const bool bit = (id >> b) & 1;
            const uint64_t bb = __ballot(bit);
            m &= bit ? bb : ~bb;
        }
        if (valid) {
            const int32_t rank = __popcll(m & ((1ull << lane) - 1ull));
            const int32_t pos = wbase[id] + rank;
            const bool leader = (m >> lane) == 1ull;   // highest lane of the group
            if (leader) wbase[id] = pos + 1;
            a.perm[pos] = (int32_t)p;
            a.inv_perm[p] = pos;
            a.row_token[pos] = (int32_t)((uint32_t)p / (uint32_t)a.K);
        }
    }
}

// Whole pack step in one workgroup, for calls of at most kPackFusedMax pairs
// (decode batches): histogram, scans, work lists and stable ranks without
// leaving LDS, and no separate clear of the error word.  16 wavefronts; wave w
// owns the consecutive pairs [w*sub, (w+1)*sub) and keeps them in registers.
constexpr int kPackFusedMax = 4096;
__device__ __forceinline__ void pack_fused(const PackArgs &a, int nbits, int32_t *lds)
{
    // lds: wbase[16][E], then wave_tot5[16][5], err
    int32_t (*wave_tot5)[5] = (int32_t (*)[5])(lds + 16 * a.E);
    int32_t *lerr = lds + 16 * a.E + 80;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int kIter = kPackFusedMax / 1024;   // 64-pair groups per wave
    for (int i = threadIdx.x; i < 16 * a.E; i += 1024) lds[i] = 0;
    if (threadIdx.x == 0) *lerr = 0;
    const int64_t start = (int64_t)wave * (kIter * 64);
    int32_t id[kIter];
    bool bad = false;
#pragma unroll
    for (int it = 0; it < kIter; ++it) {
        const int64_t p = start + it * 64 + lane;
        id[it] = p < a.P ? a.ids[p] : -1;
        if (p < a.P && (uint32_t)id[it] >= (uint32_t)a.E) { bad = true; id[it] = -1; }
    }
    __syncthreads();
    if (bad) atomicOr(lerr, 1);
#pragma unroll
    for (int it = 0; it < kIter; ++it)
        if (id[it] >= 0) atomicAdd(&lds[wave * a.E + id[it]], 1);
    __syncthreads();
    const int e = threadIdx.x;
    int32_t total = 0;
    if (e < a.E) {
        for (int w = 0; w < 16; ++w) total += lds[w * a.E + e];
        a.counts[e] = total;
        if (a.activation) a.activation[e] += (uint64_t)total;
        if (total > 0 && a.slabs != nullptr && a.slabs[e].upgate == nullptr) atomicOr(lerr, 2);
    }
    // offsets and the four lists' positions in one scan
    const SegmentCut c = cut_segment(total, a.lists.one_class);
    const int32_t v5[5] = {total, c.n128, c.n64, c.n32, c.ns};
    int32_t ex[5], tot5[5];
    block_exclusive_scan5(v5, wave_tot5, ex, tot5);
    const int32_t off = ex[0];
    if (e < a.E) {
        a.offsets[e] = off;
        int32_t run = off;
        for (int w = 0; w < 16; ++w) {
            const int32_t t = lds[w * a.E + e];
            lds[w * a.E + e] = run;
            run += t;
        }
    }
    if (e == 0) a.offsets[a.E] = tot5[0];
    if (a.lists.count != nullptr) {
        if (e < a.E && total > 0) emit_items(a.lists, e, off, total, ex[1], ex[2], ex[3], ex[4]);
        if (e == 0) {
            a.lists.count[kListT128] = tot5[1];
            a.lists.count[kListT64] = tot5[2];
            a.lists.count[kListT32] = tot5[3];
            a.lists.count[kListStream] = tot5[4];
            if (a.tile_items_host) *a.tile_items_host = tot5[1] + tot5[2] + tot5[3];
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) a.err[0] = *lerr;
#pragma unroll
    for (int it = 0; it < kIter; ++it) {
        const int64_t p = start + it * 64 + lane;
        const bool valid = id[it] >= 0;
        if (p < a.P && !valid) a.inv_perm[p] = -1;
        uint64_t m = __ballot(valid);
        for (int b = 0; b < nbits; ++b) {
            const bool bit = (id[it] >> b) & 1;
            const uint64_t bb = __ballot(bit);
            m &= bit ? bb : ~bb;
        }
        if (valid) {
            const int32_t rank = __popcll(m & ((1ull << lane) - 1ull));
            const int32_t pos = lds[wave * a.E + id[it]] + rank;
            const bool leader = (m >> lane) == 1ull;
            if (leader) lds[wave * a.E + id[it]] = pos + 1;
            a.perm[pos] = (int32_t)p;
            a.inv_perm[p] = pos;
            a.row_token[pos] = (int32_t)((uint32_t)p / (uint32_t)a.K);
        }
    }
}

__global__ __launch_bounds__(1024) void pack_fused_kernel(PackArgs a, int nbits)
{
    extern __shared__ int32_t pack_lds[];
    pack_fused(a, nbits, pack_lds);
}

// Workgroup 0 packs, the others quantise 16 rows each, one wave a row.
template <typename T>
__global__ __launch_bounds__(1024) void pack_quant_kernel(PackArgs a, int nbits)
{
    extern __shared__ int32_t pack_lds[];
    if (blockIdx.x == 0) {
        pack_fused(a, nbits, pack_lds);
        return;
    }
    typedef T V8 __attribute__((ext_vector_type(8)));
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)(blockIdx.x - 1) * 16 + (threadIdx.x >> 6);
    if (row >= a.quant_T) return;
    const V8 *x = (const V8 *)((const T *)a.quant_x + row * a.quant_H);
    uint32_t mb = 0;
    for (int c = lane; c < a.quant_H / 8; c += 64) {
        const V8 v = x[c];
#pragma unroll
        for (int j = 0; j < 8; ++j) mb = max(mb, __builtin_bit_cast(uint32_t, (float)v[j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, d));
    const QuantRow q(__builtin_bit_cast(float, mb));
    for (int c = lane; c < a.quant_H / 8; c += 64) {
        const V8 v = x[c];
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
        *(uint2 *)(a.quant_q + row * a.quant_H + c * 8) = q.codes(f);
    }
    if (lane == 0) a.quant_scale[row] = q.scale();
}

bool launch_pack(const PackArgs &a, hipStream_t s)
{
    if (a.P <= 0) {
        // offsets and counts must still be defined (all zero)
        PackArgs z = a;
        z.nblocks = 0;
        z.P = 0;
        hipLaunchKernelGGL(pack_scan_kernel, dim3(1), dim3(1024), 0, s, z);
        return false;
    }
    int nbits = 0;
    while ((1 << nbits) < a.E) ++nbits;
    // the one-workgroup form keeps 16 histograms in dynamic LDS: up to 64 KiB of it (E <= 1018).
    // (One workgroup for longer calls was measured and is slower, 85 against 43 us at 65536 pairs:
    // a single CU's memory pipeline then takes every scattered store of perm and row_token.)
    const size_t lds_bytes = sizeof(int32_t) * (16 * (size_t)a.E + 96);
    if (a.P <= kPackFusedMax && lds_bytes <= 65536) {
        if (a.quant_x) {
            const dim3 grid((unsigned)(1 + (a.quant_T + 15) / 16));
            if (a.quant_act == 0) hipLaunchKernelGGL(pack_quant_kernel<__bf16>, grid, dim3(1024), lds_bytes, s, a, nbits);
            else hipLaunchKernelGGL(pack_quant_kernel<_Float16>, grid, dim3(1024), lds_bytes, s, a, nbits);
            return true;
        }
        hipLaunchKernelGGL(pack_fused_kernel, dim3(1), dim3(1024), lds_bytes, s, a, nbits);
        return false;
    }
    hipLaunchKernelGGL(pack_hist_kernel, dim3(a.nblocks), dim3(kPackThreads), 0, s, a);
    hipLaunchKernelGGL(pack_scan_kernel, dim3(1), dim3(1024), 0, s, a);
    hipLaunchKernelGGL(pack_rank_kernel, dim3(a.nblocks), dim3(kRankThreads), sizeof(int32_t) * (kRankThreads / 64) * (size_t)a.E, s, a, nbits);
    return false;
}

// Xp[j, :] = x[row_token[j], :], 16 bytes per lane, one workgroup per row slice.
__global__ __launch_bounds__(256) void gather_rows_kernel(const uint4 *x, const int32_t *row_token,
                                                         int64_t P, int64_t row_vec, uint4 *xp)
{
    const int64_t j = blockIdx.y;
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= P || c >= row_vec) return;
    xp[j * row_vec + c] = x[(int64_t)row_token[j] * row_vec + c];
}

void launch_gather(const void *x, const int32_t *row_token, int64_t P, int64_t row_bytes, void *xp,
                   hipStream_t s)
{
    if (P <= 0) return;
    const int64_t row_vec = row_bytes / 16;
    // grid.y is limited to 65535: walk P in slabs
    for (int64_t j0 = 0; j0 < P; j0 += 65535) {
        const int64_t nj = (P - j0) < 65535 ? (P - j0) : 65535;
        hipLaunchKernelGGL(gather_rows_kernel, dim3((row_vec + 255) / 256, nj), dim3(256), 0, s,
                           (const uint4 *)x, row_token + j0, nj, row_vec,
                           (uint4 *)xp + j0 * row_vec);
    }
}

}  // namespace ek
