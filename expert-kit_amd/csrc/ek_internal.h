// Internal declarations shared by the HIP kernels and the C-ABI host code.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ek {

// ---- HBM weight layout ------------------------------------------------------
// A weight matrix [N, K] (row-major, out_features x in_features) is stored as
// 1 KiB chunks.  One chunk is what one wavefront fetches with a single 16-byte
// load per lane and feeds to MFMA without any shuffle:
//   chunk (nt, kt) covers rows nt*16 .. nt*16+15 and KE consecutive k
//   (KE = 64 for int8, 32 for 16-bit types); lane l = g*16 + i holds the
//   16 bytes W[nt*16 + i][kt*KE + g*KE/4 .. + KE/4).
// A "matrix group" interleaves NMAT matrices of equal shape chunk by chunk
// (up and gate are one group, so one wave streams one contiguous range):
//   byte offset of chunk (nt, kt, m) = ((nt*KT + kt)*NMAT + m) * 1024.
// int8 values are stored offset-binary (q + 128, i.e. q ^ 0x80) so that
// v_cvt_f32_ubyte* converts them; the kernels fold the -128 into the
// dequantisation fma.
constexpr int kChunkBytes = 1024;

// How a layer keeps its weights in HBM.
enum WeightMode {
    kW16 = 0,        // the activation type (bf16 / fp16): 32 contraction elements per 1 KiB chunk
    kWI8 = 1,        // int8, offset-binary, one fp32 scale per output channel: 64 per chunk
    kWF8Block = 2,   // fp8 e4m3fn, one fp32 scale per 128 x 128 block: 64 per chunk
    kWI8Block = 3    // int8, offset-binary, one fp32 scale per 128 x 128 block: 64 per chunk
};
constexpr bool block_scaled(int wm) { return wm == kWF8Block || wm == kWI8Block; }

struct ExpertSlab {           // device addresses of one expert's tensors
    const uint8_t *upgate;    // matrix group {up, gate}: N = I, K = H
    const uint8_t *down;      // matrix group {down}:     N = H, K = I
    const float *s_up;        // fp32 scales: [I] per channel (kWI8), [ceil(I/128), ceil(H/128)] per block
    const float *s_gate;      //   (kWF8Block, kWI8Block), nullptr for 16-bit weights; same shape as s_up
    const float *s_down;      // [H] per channel, [ceil(H/128), ceil(I/128)] per block
};

// ---- work lists ---------------------------------------------------------------
// The pack step cuts every expert segment into work items for the FFN kernels:
// as many full 128-row tiles as fit, then the remainder r by size:
//   r <= 16 -> one weight-streaming item, r <= 32 / <= 64 / <= 128 -> one MFMA
//   tile of 32 / 64 / 128 rows.
// Items of one class are stored expert-ascending, rows ascending.  List sizes
// depend on the routing, list capacities only on P, so grids are fixed on the
// host and kernels drop items beyond the device-side count.
//
// Wide cut (per-expert entry points only, decided on the host): when a call's tile items
// would occupy a small part of the chip (see wide_cut_pays), every segment is cut into
// weight-streaming items of up to kWideRows rows instead and the tile lists stay empty.
struct WorkItem {
    int32_t expert;
    int32_t row0;    // first packed position
    int32_t nrows;
    int32_t pad;
};
enum { kListStream = 0, kListT32 = 1, kListT64 = 2, kListT128 = 3, kNumLists = 4 };
struct WorkLists {
    WorkItem *items[kNumLists];
    int32_t *count;              // [kNumLists]
    // 1: a segment of more than 16 rows goes into the 128-row list whole, in as few items of at most kQ8Rows rows as
    // hold it, cut evenly in blocks of 32 rows (layers on 8-bit activations, whose tile kernel takes 1 .. kQ8Rows rows);
    // 2: every segment does, however short; 3: every segment into the streaming list, in items of up to kWideRows rows
    int32_t one_class = 0;
};
constexpr int kWideRows = 64;
constexpr int kQ8Rows = 256;
// tile_items: work items the ordinary cut would give the tile kernel; one of them spreads
// over ceil(inter / 128) workgroups in stage 1 (the tile kernel's narrow form, which such calls
// get), and below half a chip of them the call takes as long as one tile's two contractions
// however few rows it has: ~30 us + (hidden + inter) x 13.6 ns, with one-byte and 16-bit weights
// alike.  The streaming kernel spreads every item over inter / 16 workgroups, each of which reads
// its item's rows, and its time grows with the rows: ~ rows x (53 ns + hidden x inter x 14.8 fs).
// Fitted on MI355X to one DeepSeek-V3 expert (hidden 7168, inter 2048; tiled 152-158 us from 64 to
// 1024 rows with int8 weights, 150 us with bf16; streamed 143 / 188 / 199 us at 512 / 640 / 768
// rows) and to the Qwen3 shape (2048, 768: tiled 66 us fp16, 69 us int8; streamed 37 / 46 / 62 us
// at 512 / 640 / 768 rows).
inline double tile_call_us(int64_t hidden, int64_t inter) { return 30.0 + (double)(hidden + inter) * 0.0136; }
inline bool wide_cut_pays(int64_t tile_items, int64_t rows, int64_t hidden, int64_t inter)
{
    if (tile_items <= 0 || tile_items * ((inter + 255) / 256) >= 128) return false;
    const double streamed_us = (double)rows * (0.053 + 1.48e-8 * (double)hidden * (double)inter);
    return streamed_us < 0.92 * tile_call_us(hidden, inter);
}
inline int64_t list_capacity(int list, int64_t P, int64_t E, int one_class = 0)
{
    if (one_class == 3) return list == kListStream ? P / kWideRows + (P < E ? P : E) : 0;
    if (one_class && list == kListT128) {
        const int64_t segments = one_class == 2 ? P : P / 17;
        return P / kQ8Rows + (segments < E ? segments : E);
    }
    if (one_class && (list != kListStream || one_class == 2)) return 0;
    const int64_t min_rows[kNumLists] = {1, 17, 33, 65};
    const int64_t by_rows = P / min_rows[list];
    if (list == kListT128) return by_rows;
    return by_rows < E ? by_rows : E;
}

// How a layer call of P pairs on 8-bit activations is cut (WorkLists::one_class), measured on MI355X:
//  * 3, a small call on a layer whose weights fit the caches, which is bound by its launches (16 experts of 1024 x 512, top-2,
//    64 / 512 tokens: 28.5 / 40 us against 32 / 47 with tile launches beside the streaming ones; with weights beyond the
//    caches the streaming kernel's short form is better: 128 experts of 2048 x 768, 64 tokens 150 against 137 us);
//  * 2, from 16 pairs per expert on: most segments are longer than the streaming kernel's 16 rows, and a streaming
//    launch that finds little costs more than the few short tiles (DeepSeek-V3 shape, 512 / 1024 / 2048 tokens: 1905 / 1996 /
//    2140 us against 2040 / 2066 / 2200; Qwen3 shape, 256 / 1024 tokens: 152 / 210 against 157 / 225);
//  * 1 otherwise.
inline int q8_one_class(int64_t P, int64_t E, int64_t hidden, int64_t inter)
{
    if (P <= 1024 && E * 3 * hidden * inter <= (64ll << 20)) return 3;
    return P >= 16 * E ? 2 : 1;
}
// Estimates of one int8 product of n rows (n > 16) with N channels of K elements, by the streaming and by the tile kernel:
// the first does ~0.75 POP/s whatever the size, the second up to 2.3 but takes a round of at least one tile's
// contraction for every 256 tiles.  Fitted on MI355X: 512 rows x 7168 x 2048 24 / 84 us, 1024 x 7168 x 2048 43 / 84, 1024 x
// 7168 x 4096 82 / 85, 1024 x 2048 x 7168 47 / 36, 2048 x 7168 x 2048 80 / 85, 256 x 2048 x 7168 18 / 32.
inline double q8_stream_us(int64_t n, int64_t K, int64_t N) { return 5.0 + 2e-6 * (double)n * (double)K * (double)N / 750.0; }
inline double q8_tiles_us(int64_t items, int64_t item_rows, int64_t K, int64_t N)
{
    const int64_t rounds = (items * ((N + 255) / 256) + 255) / 256;
    const double blocks = (double)((item_rows < kQ8Rows ? item_rows : kQ8Rows) + 31) / 32.0;
    return (double)rounds * (14.0 + (double)(K + 127) / 128.0 * (0.45 + 0.1 * blocks));
}
inline double q8_tile_us(int64_t n, int64_t K, int64_t N) { return q8_tiles_us((n + kQ8Rows - 1) / kQ8Rows, n, K, N); }
// One expert's call: its rows, and how many tile items of at most item_rows rows they would be: whether both stages are
// better streamed.
inline bool q8_wide_cut_pays(int64_t rows, int64_t items, int64_t item_rows, int64_t hidden, int64_t inter)
{
    return items > 0 && q8_stream_us(rows, hidden, 2 * inter) + q8_stream_us(rows, inter, hidden) <
                            q8_tiles_us(items, item_rows, hidden, 2 * inter) + q8_tiles_us(items, item_rows, inter, hidden);
}
// Item i of the one-class cut of a segment of n rows (n > 16) into `items`: its first row and its rows.
constexpr int q8_items(int n) { return (n + kQ8Rows - 1) / kQ8Rows; }
// A grouped launch of several experts' calls: either all of them streamed in items of up to kWideRows rows, or those
// of more than 16 rows as tiles behind a streaming launch of the others (a stage's two launches run in turn).  Streaming
// reads an expert's weights once per 32 rows, at 6.5 TB/s whatever the products take, and costs a short call 9 % more than
// the short form.  Measured on MI355X, each launch on other experts than the one before, streamed / tiles beside streams, us:
//   7168 x 2048:  1 call of 40 rows 48 / 82, 1 of 500 102 / 152, 4 of 20 80 / 99, 4 of 100 168 / 146, 16 of 40 318 / 198;
//                 16 calls of 1 row with one of 200 267 / 310, with 4 of 100 285 / 253; 40 calls of 8 rows with one of 20 357 / 372
//   2048 x 768:   1 call of 40 rows 35 / 45, 4 of 100 61 / 78, 16 of 40 71 / 71; 40 calls of 8 rows with one of 200 108 / 148
// Of 119 drawn batches on four shapes (1024 x 512 to 7168 x 2048) the rule took the form more than 5 % slower in none.
struct Q8Batch {
    int64_t shorts = 0;                                          // calls of up to 16 rows
    int64_t rows = 0, tiles = 0, longest = 0, passes = 0;        // of the others
    void add(int64_t n)
    {
        if (n <= 16) { shorts += n > 0; return; }
        rows += n;
        tiles += q8_items((int)n);
        longest = n > longest ? n : longest;
        passes += n / kWideRows * (kWideRows / 32) + (n % kWideRows + 31) / 32;
    }
    bool streamed(int64_t hidden, int64_t inter) const
    {
        if (rows == 0) return false;
        const double weights_us = 3.0 * (double)hidden * (double)inter / 6.5e6;
        const double products = q8_stream_us(rows, hidden, 2 * inter) + q8_stream_us(rows, inter, hidden);
        const double reads = (double)passes * weights_us;
        return (products > reads ? products : reads) + 0.09 * (double)shorts * weights_us <
               q8_tiles_us(tiles, longest, hidden, 2 * inter) + q8_tiles_us(tiles, longest, inter, hidden);
    }
};
__host__ __device__ inline void q8_item(int n, int items, int i, int *first, int *rows)
{
    const int blocks = (n + 31) >> 5, base = blocks / items, more = blocks % items;
    const int b0 = i * base + (i < more ? i : more);
    *first = b0 * 32;
    const int end = (b0 + base + (i < more)) * 32;
    *rows = (end < n ? end : n) - *first;
}

// ---- router (logits -> ids, gate weights) -------------------------------------
struct RouterArgs {
    const void *logits;       // [T, E]
    int32_t logits_dt;        // 0 bf16, 1 f16, 2 f32
    const float *bias;        // [E] or nullptr (kind 4: added to the scores for the choice only)
    int64_t T;
    int32_t E, K;
    int32_t kind;             // ek_router_kind
    int32_t renorm;
    int32_t n_group, topk_group;
    int32_t mask_neg_inf;     // kind 4: experts outside the kept groups compete with -inf instead of 0
    float routed_scaling;
    int32_t *ids;             // [T, K]
    void *w;                  // [T, K]
    int32_t w_dt;             // 0 bf16, 1 f16, 2 f32
};
// needs E <= 1024, K <= 64, n_group <= 64 (checked by the caller)
hipError_t launch_router(const RouterArgs &a, hipStream_t s);

// ---- routing (pack) ---------------------------------------------------------
struct PackArgs {
    const int32_t *ids;       // [P]
    int64_t P;
    int32_t E;
    int32_t K;
    int32_t nblocks;          // ceil(P / kPackChunk)
    const ExpertSlab *slabs;  // [E]; upgate == nullptr means "not loaded"
    int32_t *block_hist;      // [nblocks][E]
    int32_t *counts;          // [E]
    int32_t *offsets;         // [E+1]
    int32_t *perm;            // [P]
    int32_t *inv_perm;        // [P]
    int32_t *row_token;       // [P]  perm[j] / K
    int32_t *err;             // bit 0: id out of range, bit 1: expert not loaded
    uint64_t *activation;     // [E] running sum of counts over calls, or nullptr
    int32_t *tile_items_host; // pinned host word that receives the number of tile items cut, or nullptr
    WorkLists lists;
    // 16-bit rows to quantise beside the routing (see launch_pack), or nullptr
    const void *quant_x = nullptr;      // [quant_T, quant_H], quant_H a multiple of 64
    int64_t quant_T = 0;
    int32_t quant_H = 0, quant_act = 0;
    uint8_t *quant_q = nullptr;
    float *quant_scale = nullptr;
};
constexpr int kPackChunk = 4096;   // pairs per workgroup
constexpr int kPackThreads = 256;
constexpr int kMaxExperts = 1024;

// writes *err itself (one kernel of every pack stores the call's word: nothing to clear first,
// no memset node: graph-capture safe)
// Returns whether the rows of a.quant_x have been quantised on the way: the one-workgroup form of the step leaves the
// chip idle, and further workgroups of the same launch take the rows.
bool launch_pack(const PackArgs &a, hipStream_t s);
// work lists for one segment [0, n) of expert e (per-expert forward)
void launch_single_lists(const WorkLists &lists, int32_t expert, int32_t n, bool wide, hipStream_t s);
// lists that hold the one segment (expert, rows row0 .. row0+n-1) and nothing else; mode 0: the usual
// cut, 1: 16-row streaming items, 2: streaming items of up to kWideRows rows.  row_token, if given,
// receives row0 + t -> t.
void launch_segment_lists(const WorkLists &lists, int32_t expert, int32_t row0, int32_t n, int32_t *row_token, int mode,
                          hipStream_t s);
// appends the segment (expert, rows row0 .. row0+n-1) to the lists pack has built and maps
// its rows to tokens 0 .. n-1.  as_stream: 0 the usual cut; 1 all rows as 16-row streaming items;
// 2 all rows as streaming items of up to kWideRows rows, which replace the streaming list (the
// caller passes a list of their own)
void launch_append_segment(const WorkLists &lists, int32_t expert, int32_t row0, int32_t n, int32_t *row_token,
                           int as_stream, hipStream_t s);
void launch_gather(const void *x, const int32_t *row_token, int64_t P, int64_t row_bytes, void *xp,
                   hipStream_t s);

// ---- grouped FFN -------------------------------------------------------------
struct FfnArgs {
    const void *x;            // activations, row stride x_stride elements
    int64_t x_stride;
    const int32_t *rows;      // packed position -> row of x, or nullptr (identity)
    const ExpertSlab *slabs;  // [E]
    void *out;                // stage 1: h [P, N]; stage 2: yp [P, N]
    int64_t out_stride;
    int32_t N;                // output channels of this stage
    int32_t Kdim;             // contraction length of this stage
    WorkLists lists;          // device work lists and their lengths
    // pair-direct launches (launch_ffn_pairs): pair p = t * pair_K + k is its own one-row item,
    // x row t (stage 1) or p (stage 2), out row p; no lists
    const int32_t *pair_ids = nullptr;   // [pair_P] expert of pair p
    int32_t pair_K = 0, pair_P = 0, n_experts = 0;
    const void *pair_w = nullptr;        // [pair_P] gate weights (stage 2)
    int32_t pair_w_f32 = 0;              // gate weights are fp32 instead of the activation type
    int32_t pair_shared = 0;             // 1: every token also runs expert n_experts (the shared expert) as item
                                         // pair_P + t (x row t, out row pair_P + t); its rounded output is added
                                         // to the rounded weighted sum, as the combine kernel adds it
    void *pair_y = nullptr;              // [T, N] stage 2: the weighted sum over a token's pairs
    int32_t *pair_err = nullptr;         // stage 1 writes the call's error word (PackArgs::err)
    uint64_t *pair_activation = nullptr; // [n_experts] or nullptr (PackArgs::activation)
    int32_t *pair_tile_items_host = nullptr;   // receives 0 (PackArgs::tile_items_host), or nullptr
};
// Most pairs a pair-direct call may hold (one wave writes the call's bookkeeping) and its
// largest top-k (one wave per pair of a token in stage 2's workgroups).
constexpr int kPairDirectMax = 64, kPairDirectMaxK = 8;
// A decode call of a few pairs without pack and combine kernels: stage 1 runs every pair as a
// one-row item straight from the ids (and stores what the pack kernel would have stored of the
// call's bookkeeping: error word, activation counters, zero tile items); stage 2 computes a
// token's pairs in one workgroup, one wave each, and adds them in k order with the gate weights:
// the arithmetic of the streaming kernel followed by launch_combine, bit for bit.  Pairs whose
// id is out of range or whose expert is not loaded add nothing.  T = pair_P / pair_K.
hipError_t launch_ffn_pairs(const FfnArgs &a, int stage, int act, int wmode, hipStream_t s);
// stage = 1: up/gate + SwiGLU epilogue;  stage = 2: down projection
// act: 0 bf16, 1 f16;  wmode: WeightMode
// weight-streaming kernel over lists.items[kListStream]; max_items = grid bound;
// wide: items hold up to kWideRows rows (else up to 16); few_rows: about four rows or fewer per
// item on average (a hint for the launch shape; the results do not depend on it)
hipError_t launch_ffn_stream(const FfnArgs &a, int stage, int act, int wmode, int64_t max_items, bool wide,
                             bool few_rows, hipStream_t s);
// MFMA tile kernel over the three tile lists (128-row items first, then 64,
// then 32); max_items[l] bounds list l.  A workgroup covers tile_channels(stage, narrow) output
// channels of one item; the narrow form (half the channels per workgroup, so twice the workgroups
// per item; same bits) is for launches that would leave most of the chip without a tile.
hipError_t launch_ffn_tile(const FfnArgs &a, int stage, int act, int wmode,
                           const int64_t max_items[kNumLists], bool narrow, hipStream_t s);
// hidden channels (stage 1) / output channels (stage 2) per tile workgroup
constexpr int tile_channels(int stage, bool narrow) { return (stage == 1 ? 256 : 512) / (narrow ? 2 : 1); }

// ---- 8-bit activations ----------------------------------------------------------
// Rows of 16-bit values -> int8 rows and one scale per row, with (norm) the residual's addition and the
// RMS norm in front: see ek_quant.hip for the definition.
struct RowQuantArgs {
    const void *x;            // [n, H] activation type
    const void *residual;     // [n, H] or nullptr (norm)
    const void *gain;         // [H] (norm)
    void *sum;                // [n, H] or nullptr: x + residual (norm)
    void *y;                  // [n, H] or nullptr: the normed rows (norm)
    uint8_t *q;               // [n, q_stride] int8 or nullptr; columns H .. q_stride-1 are set to zero
    float *scale;             // [n] or nullptr
    int64_t n;
    int32_t H;                // norm: a multiple of 8
    int32_t q_stride;         // a multiple of 8, at least H
    float eps;
    double inv_h;             // 1 / H
    bool vec;                 // rows of x start on 16-byte boundaries (H a multiple of 8)
};
hipError_t launch_row_quant(const RowQuantArgs &a, int act, bool norm, hipStream_t s);
// int8 rows of len bytes back to back -> rows of `stride` bytes with a zero tail
hipError_t launch_pad_rows8(const void *src, int64_t n, int32_t len, void *dst, int32_t stride, hipStream_t s);

// Products of int8 rows with int8 weights (per-channel scales): ek_ffn_q8.hip
struct Q8Args {
    const uint8_t *x;         // int8 rows, stride Kdim bytes
    const float *x_scale;     // one per row of x
    const int32_t *rows;      // packed position -> row of x, or nullptr (identity)
    const ExpertSlab *slabs;
    void *out;                // stage 1: h; stage 2: output rows (packed order), activation type
    int64_t out_stride;
    int32_t N;                // output channels stored (stage 1: a multiple of 16)
    int32_t NT;               // 16-channel tiles the weights hold
    int32_t Kdim;             // a multiple of 64
    const float *bias;        // [N] or nullptr (stage 2)
    WorkLists lists;          // dense calls (one matrix, rows 0 .. n-1): items[] unused
    int64_t dense_rows = 0;   // > 0: a dense call of that many rows on slab 0
};
// stage 1: up/gate + SwiGLU; stage 2: one matrix.  max_items[l]: bound of list l (see launch_ffn_tile);
// wide: the streaming list holds items of up to kWideRows rows
hipError_t launch_ffn_q8(const Q8Args &a, int stage, int act, const int64_t max_items[kNumLists], bool wide, hipStream_t s);
hipError_t launch_dense_q8(const Q8Args &a, int act, hipStream_t s);
// A decode call of a few pairs without pack, quantisation and combine kernels (as launch_ffn_pairs): up (a.x with
// x_scale, or pa.x16; out = h rows in pair order) and down (out_stride = N) stage arguments.
struct PairArgs {
    const int32_t *ids;       // [P]
    int32_t P, K, n_experts;
    int32_t shared;           // 1: every token also runs expert n_experts, rows P .. P + T - 1 of h
    const void *x16;          // 16-bit rows of x, or nullptr: 8-bit ones in the stage's arguments
    const void *h;            // stage 1's output
    const void *w;            // [P] gate weights
    int32_t w_f32;
    void *y;                  // [T, N]
    int32_t *err;             // the call's bookkeeping, as the pack kernel would store it
    uint64_t *activation;
};
// LDS holds a token's rows of h as codes (and stage 1's row of x)
inline bool q8_pairs_fit(int64_t P, int64_t K, int64_t hidden, int64_t inter)
{
    return P > 0 && P <= kPairDirectMax && K <= kPairDirectMaxK && P % K == 0 && (kPairDirectMaxK + 1) * inter <= 60 * 1024 && hidden <= 60 * 1024;
}
hipError_t launch_pairs_q8(const Q8Args &up, const Q8Args &down, const PairArgs &pa, int act, hipStream_t s);

// ---- combine ----------------------------------------------------------------
struct CombineArgs {
    const void *yp;           // [P, H] packed expert outputs
    const int32_t *inv_perm;  // [T*K]
    const void *w;            // [T, K]
    void *y;                  // [T, H]
    int64_t T;
    int32_t K;
    int64_t H;
    int32_t act;              // 0 bf16, 1 f16
    int32_t w_f32;            // gate weights are fp32 (DeepSeek shim) instead of act dtype
    const void *shared;       // [T, H] shared-expert output added to the rounded sum, or nullptr
};
void launch_combine(const CombineArgs &a, hipStream_t s);

// ---- batched row copies -----------------------------------------------------
// One launch moves the rows of many requests between the callers' buffers and a staging buffer
// (instead of one asynchronous copy per request, ~4 us of host time each).
struct RowCopy {
    const uint8_t *src;
    uint8_t *dst;
    int64_t src_pitch, dst_pitch;   // bytes from one row to the next
    int32_t rows;
    int32_t row_bytes;              // a multiple of 16; src and dst are 16-byte aligned
};
// segs: n entries the device can read (device memory or pinned host memory), unchanged until the
// kernel has run
void launch_rows_copy(const RowCopy *segs, int n, hipStream_t s);

// one wave idling for iters x ~1000 cycles (see pick_side_stream in ek_capi.hip)
void launch_idle(int iters, hipStream_t s);

// ---- weight ingestion -------------------------------------------------------
// src [N, K] row-major of src_dtype (ek_dtype numbering) -> chunked layout at
// dst, matrix m of an nmat-group.  dst_dtype: 0 bf16, 1 f16, 3 int8.  block_scale (16-bit
// destinations only, may be nullptr): [ceil(N/128), ceil(K/128)] factors of scale_dtype.
void launch_tile_weights(const void *src, int src_dtype, int64_t N, int64_t K, uint8_t *dst,
                         int dst_dtype, int m, int nmat, const void *block_scale, int scale_dtype,
                         hipStream_t s);
void launch_scales_to_f32(const void *src, int src_dtype, int64_t n, float *dst, hipStream_t s);

}  // namespace ek
