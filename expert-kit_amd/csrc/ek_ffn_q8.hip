// Products of int8 activation rows with int8 weights: the two stages of the expert FFN on 8-bit
// activations, and one matrix alone (ek_linear).
//
//   u[n, c] = sum_k q[n, k] w[c, k] * scale[n] * w_scale[c]
//
// with the integer sum exact: codes and weights are -128 .. 127 and the contraction at most 131072 long, so the
// sum lies between -127 * 128 * 131072 and 2^31 = 128 * 128 * 131072.  That one sum does not fit int32; see q8_sum.
// Integer addition is associative, so every split of the contraction and every tile shape below gives the same bits.
// Weights lie in HBM as for W8A16 (ek_internal.h): one 1 KiB chunk is the A operand of
// v_mfma_i32_16x16x64_i8 as it is, but for the offset-binary storage: q = u ^ 0x80.
#include "ek_internal.h"
#include "ek_mfma.h"
#include "ek_quant.h"

#include <type_traits>

namespace ek {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i32x4 signed8(uint4 u, uint32_t flip = 0x80808080u)
{
    return i32x4{(int)(u.x ^ flip), (int)(u.y ^ flip), (int)(u.z ^ flip), (int)(u.w ^ flip)};
}

// A sum before its conversion to fp32.  Only 2^31 wraps, to the one value that no other sum has; the largest int32
// becomes 2^31 when it is rounded to fp32.
constexpr int kQ8WrapChunks = 131072 / 64;       // only the longest contraction can reach it
__device__ __forceinline__ int q8_sum(int s) { return s == INT32_MIN ? INT32_MAX : s; }

// Four consecutive channels ch .. ch+3 of one output row.
template <typename T>
__device__ __forceinline__ void store4(T *orow, int ch, int N, bool whole, const float *v)
{
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (whole) {
        T4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = (T)v[r];
        *(uint2 *)(orow + ch) = __builtin_bit_cast(uint2, o);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (ch + r < N) orow[ch + r] = (T)v[r];
    }
}

constexpr int kQ8Slices = 8;

// One workgroup: RS*16 rows x NG*16 channels (of NMAT matrices); its eight waves take an eighth of the
// contraction each and meet in LDS.  Operands come straight from memory, D chunks ahead.
//
// Up to 16 rows (RS = 1) the call is bound by the weights: one channel tile (of up and gate) per workgroup gives the
// most loads in flight.  Longer items take RS = 2 rows of fragments x 4 chunks of weights: every fragment of the
// rows is read by N / 64 workgroups instead of N / 16, which is what the call waits for (MI355X, 64 rows of 7168 x 2048:
// 16.7 us with one tile and 64 rows, 10.9 with two tiles and 32 rows, 12.6 with four; 512 rows: 56, 35 and 24 us; 64 rows
// of 2048 x 7168: 11.4, 8.2 and 7.2 us).
template <typename T, int NMAT, int NG, int RS, int D>
__global__ __launch_bounds__(64 * kQ8Slices) void q8_stream_kernel(Q8Args a, int list, int item_rows)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = lane & 15, g = lane >> 4;
    int e = 0, seg0, n;
    if (a.dense_rows > 0) {
        const int64_t r0 = (int64_t)blockIdx.y * item_rows;
        seg0 = (int)r0;
        n = (int)min((int64_t)item_rows, a.dense_rows - r0);
    } else {
        if ((int)blockIdx.y >= a.lists.count[list]) return;
        const WorkItem item = a.lists.items[list][blockIdx.y];
        e = item.expert; seg0 = item.row0; n = item.nrows;
    }
    // part blockIdx.z of the item
    seg0 += blockIdx.z * (RS * 16);
    n = min(n - (int)blockIdx.z * (RS * 16), RS * 16);
    if (n <= 0) return;
    const int nt0 = blockIdx.x * NG;
    const ExpertSlab slab = a.slabs[e];
    const uint8_t *wmat = NMAT == 2 ? slab.upgate : slab.down;
    if (wmat == nullptr) return;             // expert not loaded: the call has been flagged
    const int KT = a.Kdim >> 6;
    const int nfr = (n + 15) >> 4;

    const uint8_t *wp[NG];
#pragma unroll
    for (int gi = 0; gi < NG; ++gi)          // tiles past the last one recompute it and store nothing
        wp[gi] = wmat + (int64_t)min(nt0 + gi, a.NT - 1) * KT * (NMAT * kChunkBytes) + lane * 16;
    const uint8_t *xp[RS];
    float xs[RS];
#pragma unroll
    for (int rs = 0; rs < RS; ++rs) {
        const int jr = min(rs * 16 + j, n - 1);
        const int64_t row = a.rows ? (int64_t)a.rows[seg0 + jr] : (int64_t)(seg0 + jr);
        xp[rs] = a.x + row * a.Kdim + g * 16;
        xs[rs] = a.x_scale[row];
    }
    i32x4 acc[RS][NMAT][NG];
#pragma unroll
    for (int rs = 0; rs < RS; ++rs)
#pragma unroll
        for (int m = 0; m < NMAT; ++m)
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) acc[rs][m][gi] = i32x4{0, 0, 0, 0};

    const int kbeg = KT * wave / kQ8Slices, kend = KT * (wave + 1) / kQ8Slices;
    uint4 wq[D][NG][NMAT], xq[D][RS];
    auto fetch = [&](int d, int kt) {
#pragma unroll
        for (int gi = 0; gi < NG; ++gi)
#pragma unroll
            for (int m = 0; m < NMAT; ++m) {
                const uint8_t *src = wp[gi] + (int64_t)(kt * NMAT + m) * kChunkBytes;
                wq[d][gi][m] = RS == 1 ? ldg16_once(src) : ldg16(src);
            }
#pragma unroll
        for (int rs = 0; rs < RS; ++rs)
            if (RS == 1 || rs < nfr) xq[d][rs] = ldg16(xp[rs] + (int64_t)kt * 64);
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (kbeg + d < kend) fetch(d, kbeg + d);
    for (int kt0 = kbeg; kt0 < kend; kt0 += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int kt = kt0 + d;
            if (kt >= kend) break;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi)
#pragma unroll
                for (int m = 0; m < NMAT; ++m) {
                    const i32x4 w = signed8(wq[d][gi][m]);
#pragma unroll
                    for (int rs = 0; rs < RS; ++rs)
                        if (RS == 1 || rs < nfr)
                            acc[rs][m][gi] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, __builtin_bit_cast(i32x4, xq[d][rs]),
                                                                                   acc[rs][m][gi], 0, 0, 0);
                }
            if (kt + D < kend) fetch(d, kt + D);
        }
    }

    // the slices' sums meet in LDS; wave w finishes fragment (rs, gi) number w, w + 8, ...
    __shared__ i32x4 red[kQ8Slices][RS * NMAT * NG][64];
#pragma unroll
    for (int rs = 0; rs < RS; ++rs)
        if (RS == 1 || rs < nfr) {
#pragma unroll
            for (int m = 0; m < NMAT; ++m)
#pragma unroll
                for (int gi = 0; gi < NG; ++gi) red[wave][(rs * NMAT + m) * NG + gi][lane] = acc[rs][m][gi];
        }
    __syncthreads();
#pragma unroll
    for (int f = 0; f < RS * NG; ++f) {
        if (f % kQ8Slices != wave) continue;
        const int rs = f / NG, gi = f % NG;
        if (rs * 16 + j >= n || nt0 + gi >= a.NT) continue;
        i32x4 tot[NMAT];
#pragma unroll
        for (int m = 0; m < NMAT; ++m) {
            tot[m] = red[0][(rs * NMAT + m) * NG + gi][lane];
#pragma unroll
            for (int w = 1; w < kQ8Slices; ++w) tot[m] += red[w][(rs * NMAT + m) * NG + gi][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) tot[m][r] = q8_sum(tot[m][r]);
        }
        // lane (g, j) holds channels 4g .. 4g+3 of row j
        const int ch = (nt0 + gi) * 16 + 4 * g;
        T *orow = (T *)a.out + (int64_t)(seg0 + rs * 16 + j) * a.out_stride;
        float v[4];
        if constexpr (NMAT == 2) {
            const float4 su = *(const float4 *)(slab.s_up + ch), sg = *(const float4 *)(slab.s_gate + ch);
            const float us[4] = {su.x, su.y, su.z, su.w}, gs[4] = {sg.x, sg.y, sg.z, sg.w};
#pragma unroll
            for (int r = 0; r < 4; ++r)
                v[r] = (float)swiglu_rounded<T>(as_fp32((float)tot[0][r] * (xs[rs] * us[r])), as_fp32((float)tot[1][r] * (xs[rs] * gs[r])));
            store4<T>(orow, ch, a.N, true, v);
        } else {
            const float4 s4 = *(const float4 *)(slab.s_down + ch);
            const float ws[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                v[r] = as_fp32((float)tot[0][r] * (xs[rs] * ws[r]));
                if (a.bias && ch + r < a.N) v[r] += a.bias[ch + r];
            }
            store4<T>(orow, ch, a.N, (a.out_stride & 3) == 0 && ch + 4 <= a.N, v);
        }
    }
}


// ---- pair-direct calls: a few (token, expert) pairs, two kernels ------------------------------------------
//
// Every pair is a one-row item taken straight from the ids, as launch_ffn_pairs does for 16-bit activations.
// Stage 1: blockIdx.y is the pair; the eight waves take an eighth of the contraction each.  With 16-bit rows of x the
// workgroup quantises its row first (into LDS).  Stage 2: blockIdx.y is the token, wave k takes its k-th pair: it
// quantises the pair's row of h into LDS, walks the whole contraction, and the first wave adds the
// rounded outputs with the gate weights in k order, as the combine kernel does.  The integer sums are exact and the codes
// are functions of their row, so the results are those of the call through pack and combine, bit for bit.

// What the pack kernel would have stored of the call's bookkeeping; one wave.
__device__ __forceinline__ void pair_bookkeeping(const PairArgs &pa, const ExpertSlab *slabs, int lane)
{
    const int32_t id = lane < pa.P ? pa.ids[lane] : 0;
    const bool bad = lane < pa.P && (uint32_t)id >= (uint32_t)pa.n_experts, ok = lane < pa.P && !bad;
    const bool unloaded = ok && slabs[id].upgate == nullptr;
    const uint64_t any_bad = __ballot(bad), any_unloaded = __ballot(unloaded);
    if (ok && pa.activation) atomicAdd((unsigned long long *)&pa.activation[id], 1ull);
    if (lane == 0) pa.err[0] = (any_bad ? 1 : 0) | (any_unloaded ? 2 : 0);
}

// The codes of one row of n 16-bit values (n a multiple of 64) by the THREADS lanes that hold it, into LDS; returns the
// scale.  red: one word per wave.
template <typename T, int WAVES>
__device__ __forceinline__ float q8_row_to_lds(const T *row, int n, uint8_t *codes, uint32_t *red)
{
    typedef T V8 __attribute__((ext_vector_type(8)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = WAVES == 1 ? lane : threadIdx.x;
    uint32_t mb = 0;
    for (int c = tid; c < n / 8; c += 64 * WAVES) {
        const V8 v = *(const V8 *)(row + c * 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) mb = max(mb, __builtin_bit_cast(uint32_t, (float)v[j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) mb = max(mb, (uint32_t)__shfl_xor((int)mb, d));
    if constexpr (WAVES > 1) {
        if (lane == 0) red[wave] = mb;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mb = max(mb, red[w]);
    }
    const QuantRow q(__builtin_bit_cast(float, mb));
    for (int c = tid; c < n / 8; c += 64 * WAVES) {
        const V8 v = *(const V8 *)(row + c * 8);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
        *(uint2 *)(codes + c * 8) = q.codes(f);
    }
    return q.scale();
}

template <typename T>
__global__ __launch_bounds__(64 * kQ8Slices) void q8_pairs_up_kernel(Q8Args a, PairArgs pa)
{
    extern __shared__ __align__(16) uint8_t q8_lds[];            // 16-bit rows: the codes of this pair's row
    __shared__ uint32_t red_m[kQ8Slices];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
    if (blockIdx.x == 0 && blockIdx.y == 0 && wave == 0) pair_bookkeeping(pa, a.slabs, lane);
    const int pair = blockIdx.y;
    const bool shared_row = pair >= pa.P;
    const int e = shared_row ? pa.n_experts : pa.ids[pair];
    if (!shared_row && (uint32_t)e >= (uint32_t)pa.n_experts) return;
    const ExpertSlab slab = a.slabs[e];
    if (slab.upgate == nullptr) return;
    const int64_t row = shared_row ? pair - pa.P : pair / pa.K;
    const int KT = a.Kdim >> 6, nt = blockIdx.x;
    const int kbeg = KT * wave / kQ8Slices, kend = KT * (wave + 1) / kQ8Slices;
    const uint8_t *wp = slab.upgate + (int64_t)nt * KT * (2 * kChunkBytes) + lane * 16;
    constexpr int D = 4;
    uint4 wq[D][2];
    auto fetch = [&](int d, int kt) {
#pragma unroll
        for (int m = 0; m < 2; ++m) wq[d][m] = ldg16_once(wp + (int64_t)(kt * 2 + m) * kChunkBytes);
    };
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (kbeg + d < kend) fetch(d, kbeg + d);
    float xs;
    if (pa.x16) xs = q8_row_to_lds<T, kQ8Slices>((const T *)pa.x16 + row * a.Kdim, a.Kdim, q8_lds, red_m);
    else xs = a.x_scale[row];
    if (pa.x16) __syncthreads();
    const uint8_t *xg = a.x + row * a.Kdim + g * 16, *xl = q8_lds + g * 16;
    i32x4 acc[2] = {i32x4{0, 0, 0, 0}, i32x4{0, 0, 0, 0}};
    for (int kt0 = kbeg; kt0 < kend; kt0 += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int kt = kt0 + d;
            if (kt >= kend) break;
            const i32x4 x = pa.x16 ? *(const i32x4 *)(xl + kt * 64) : __builtin_bit_cast(i32x4, ldg16(xg + kt * 64));
#pragma unroll
            for (int m = 0; m < 2; ++m) acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(signed8(wq[d][m]), x, acc[m], 0, 0, 0);
            if (kt + D < kend) fetch(d, kt + D);
        }
    }
    // every column of the result is the row: lanes j = 0 keep it
    __shared__ i32x4 red[kQ8Slices][2][4];
    if (j == 0) { red[wave][0][g] = acc[0]; red[wave][1][g] = acc[1]; }
    __syncthreads();
    if (threadIdx.x >= 16) return;
    const int ch = nt * 16 + threadIdx.x;
    int up = 0, gate = 0;
#pragma unroll
    for (int w = 0; w < kQ8Slices; ++w) {
        up += red[w][0][threadIdx.x >> 2][threadIdx.x & 3];
        gate += red[w][1][threadIdx.x >> 2][threadIdx.x & 3];
    }
    ((T *)a.out)[(int64_t)pair * a.out_stride + ch] =
        swiglu_rounded<T>(as_fp32((float)up * (xs * slab.s_up[ch])), as_fp32((float)gate * (xs * slab.s_gate[ch])));
}

constexpr int kPairTiles = 2;            // channel tiles of a stage-2 workgroup
template <typename T>
__global__ __launch_bounds__(64 * (kPairDirectMaxK + 1)) void q8_pairs_down_kernel(Q8Args a, PairArgs pa)
{
    extern __shared__ __align__(16) uint8_t q8_lds[];            // [waves][Kdim]: the codes of the pairs' rows of h
    __shared__ float prod[kPairDirectMaxK + 1][kPairTiles * 16];
    __shared__ int32_t valid[kPairDirectMaxK + 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
    const int64_t t = blockIdx.y;
    const bool shared_row = wave == pa.K;
    const int64_t pair = shared_row ? pa.P + t : t * pa.K + wave;
    int e = shared_row ? pa.n_experts : pa.ids[pair];
    bool live = shared_row || (uint32_t)e < (uint32_t)pa.n_experts;
    const ExpertSlab slab = a.slabs[live ? e : 0];
    live = live && slab.down != nullptr;
    const int nt0 = blockIdx.x * kPairTiles;
    if (lane == 0) valid[wave] = live;
    if (live) {
        const int KT = a.Kdim >> 6;
        const uint8_t *wp[kPairTiles];
#pragma unroll
        for (int gi = 0; gi < kPairTiles; ++gi) wp[gi] = slab.down + (int64_t)min(nt0 + gi, a.NT - 1) * KT * kChunkBytes + lane * 16;
        constexpr int D = 4;
        uint4 wq[D][kPairTiles];
        auto fetch = [&](int d, int kt) {
#pragma unroll
            for (int gi = 0; gi < kPairTiles; ++gi) wq[d][gi] = ldg16_once(wp[gi] + (int64_t)kt * kChunkBytes);
        };
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (d < KT) fetch(d, d);
        uint8_t *codes = q8_lds + (int64_t)wave * a.Kdim;
        const float hs = q8_row_to_lds<T, 1>((const T *)pa.h + pair * a.Kdim, a.Kdim, codes, nullptr);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        i32x4 acc[kPairTiles];
#pragma unroll
        for (int gi = 0; gi < kPairTiles; ++gi) acc[gi] = i32x4{0, 0, 0, 0};
        for (int kt0 = 0; kt0 < KT; kt0 += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int kt = kt0 + d;
                if (kt >= KT) break;
                const i32x4 x = *(const i32x4 *)(codes + kt * 64 + g * 16);
#pragma unroll
                for (int gi = 0; gi < kPairTiles; ++gi)
                    acc[gi] = __builtin_amdgcn_mfma_i32_16x16x64_i8(signed8(wq[d][gi]), x, acc[gi], 0, 0, 0);
                if (kt + D < KT) fetch(d, kt + D);
            }
        }
        if (j == 0) {
            const int64_t wi = shared_row ? 0 : pair;
            const float gw = pa.w_f32 ? ((const float *)pa.w)[wi] : (float)((const T *)pa.w)[wi];
#pragma unroll
            for (int gi = 0; gi < kPairTiles; ++gi)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int ch = min((nt0 + gi) * 16 + 4 * g + r, a.NT * 16 - 1);
                    float v = (float)(T)as_fp32((float)acc[gi][r] * (hs * slab.s_down[ch]));
                    if (!shared_row) {
                        v = as_fp32(gw * v);
                        if (!pa.w_f32) v = (float)(T)v;
                    }
                    prod[wave][gi * 16 + 4 * g + r] = v;
                }
        }
    }
    __syncthreads();
    if (threadIdx.x >= kPairTiles * 16 || nt0 * 16 + (int)threadIdx.x >= a.N) return;
    float sum = 0.f;
    for (int k = 0; k < pa.K; ++k)
        if (valid[k]) sum = sum + prod[k][threadIdx.x];
    T o = (T)sum;
    if (pa.shared && valid[pa.K]) o = (T)((float)o + prod[pa.K][threadIdx.x]);       // after the sum's rounding
    ((T *)pa.y)[t * a.out_stride + nt0 * 16 + threadIdx.x] = o;
}

// ---- tile kernel: items of up to 256 rows -------------------------------------------------------------
//
// One workgroup of four wavefronts, one per SIMD: RB*32 rows x 4*64 matrix channels (stage 1: 128 hidden
// channels, up and gate of each); every wave keeps all the rows and 64 channels (256 rows: 256
// accumulator registers).  MFMA 32x32x32 i8, weights as the A operand.  Steps of 128 contraction elements:
//   - weights go from memory straight into registers, no other wave wants them: a 16-byte load per lane
//     from the chunked layout is an A operand.  A step's registers are loaded again as soon as they have been
//     used, for the third step after it;
//   - the rows' bytes are shared by the four waves: LDS-DMA into three stages (three steps ahead), rows of
//     128 bytes whose 16-byte pieces are XOR-swizzled so that fragment reads are conflict free.
// Per step of 256 rows and workgroup the vector L1 moves 64 KiB and the LDS 160 KiB against 2048 cycles of MFMA: half of
// what the one and 60 % of what the other can.  (128 rows per wave, two workgroups per CU, wants 96 KiB of the L1: it was
// the bound.  8192 x 8192 x 8192 on MI355X: 1.84 POP/s, and 2.73 with the weight loads taken out.)
// Measured on MI355X: that product 468 us = 2.35 POP/s; 8192 tokens of 256 experts of 7168 x 2048, top-8: 2.3 + 1.5 ms, the
// matrix pipes busy for 44 and 36 % of the cycles at 1.8 GHz.  With 256 tiles of 256
// rows at once a step takes 1.7 us and a tile 16 us beside its steps (launch, first loads, conversion, stores), 21 with SwiGLU, which
// is what bounds short contractions (768: two thirds of the time).
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ void dma16(const void *gaddr, uint32_t lds_addr)     // lane l's 16 bytes land at lds_addr + 16 l
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(gaddr), "s"(lds_addr) : "memory");
}
__device__ __forceinline__ void dma4(const void *gaddr, uint32_t lds_addr)      // lane l's 4 bytes at lds_addr + 4 l
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(gaddr), "s"(lds_addr) : "memory");
}
template <int N> __device__ __forceinline__ void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }
// The wave has its LDS reads back before it lets the others overwrite what it read.
__device__ __forceinline__ void block_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

constexpr int kQ8Waves = 4, kQ8Stages = 3;
constexpr int kQ8Stage = kQ8Rows * 128;                   // bytes of a stage: 256 rows x 128 elements
constexpr int kQ8ScratchPitch = 64 * 2 + 16;              // epilogue: 32 rows x 64 channels of a wave
constexpr int kQ8Scratch = 32 * kQ8ScratchPitch;
constexpr int kQ8Scales = kQ8Stages * kQ8Stage + kQ8Waves * kQ8Scratch;   // then the scales: rows, channels, bias
constexpr int kQ8Lds = kQ8Scales + 3 * 256 * 4;
static_assert(kQ8Rows == 64 * kQ8Waves && 4 * 64 == 64 * kQ8Waves, "one row and one channel scale per thread");

__device__ __forceinline__ int q8_key(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// (what names the tile is the same for every lane: scalar loads)
typedef const __attribute__((address_space(4))) int32_t *ConstInts;
typedef const __attribute__((address_space(4))) uint64_t *ConstWords;

// slab_at: the expert's ExpertSlab.  It and the rows' numbers are asked for together.
// WRAP: sums may be 2^31 (see q8_sum).  They are counted from -1 and the last addition saturates: one operation per sum,
// in an instance of its own (a selection as q8_sum's spills registers; the ordinary contraction needs neither).
template <typename T, int NMAT, int RB, bool WRAP>
__device__ __forceinline__ void q8_tile(const Q8Args &a, ConstWords slab_at, int row0, int n, int cblock, uint8_t *lds)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, kh = lane >> 5, j = lane & 15;
    const int KT = a.Kdim >> 6, nfull = KT >> 1, ns = (KT + 1) >> 1;
    // the rows' numbers in x: of thread tid's scale, and of the DMAs (instruction q brings rows 8q .. 8q+7, lane l piece
    // (l & 7) ^ key of row 8q + l / 8); rows past the item re-read its last one
    int32_t row_sc = row0 + min(tid, n - 1), row[RB];
#pragma unroll
    for (int i = 0; i < RB; ++i) row[i] = row0 + min((wave * RB + i) * 8 + (lane >> 3), n - 1);
    if (a.rows) {
        row_sc = a.rows[row_sc];
#pragma unroll
        for (int i = 0; i < RB; ++i) row[i] = a.rows[row[i]];
    }
    const ExpertSlab slab{(const uint8_t *)slab_at[0], (const uint8_t *)slab_at[1], (const float *)slab_at[2], (const float *)slab_at[3],
                          (const float *)slab_at[4]};
    const uint8_t *wmat = NMAT == 2 ? slab.upgate : slab.down;
    if (wmat == nullptr) return;                                 // expert not loaded: the call has been flagged
    const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    constexpr int kStep = 2 * NMAT * kChunkBytes;            // bytes from one step's weights to the next's
    // the wave's first 16-channel tile; block cb: matrix cb of tiles nt0, nt0 + 1, or tiles nt0 + 2 cb, + 1
    const int nt0 = (cblock * kQ8Waves + wave) * (NMAT == 2 ? 2 : 4);
    const uint8_t *wp[2];
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
        const int nt = min(nt0 + (NMAT == 2 ? 0 : cb * 2) + (l32 >> 4), a.NT - 1);   // tiles past the last recompute it
        wp[cb] = wmat + ((int64_t)nt * KT * NMAT + (NMAT == 2 ? cb : 0)) * kChunkBytes + (kh * 16 + j) * 16;
    }
    const int bkey = q8_key(l32);
    int boff[4];
#pragma unroll
    for (int kg = 0; kg < 4; ++kg) boff[kg] = l32 * 128 + ((kg * 2 + kh) ^ bkey) * 16;

    i32x16 acc[RB][2];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[rb][cb][r] = WRAP ? -1 : 0;

    constexpr int D = kQ8Stages;
    uint4 w[D][4][2];
    // one k-group's weights of the step wp points to; hi: from there to the step's second chunk
    auto load_w = [&](int slot, int kg, int hi) {
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) w[slot][kg][cb] = ldg16(wp[cb] + (kg >= 2 ? hi : 0) + (kg & 1) * 512);
    };
    // wp moves on to step s (which stays the last one where there is no step s); returns its `hi`
    auto move_w = [&](int s) {
        const int adv = s < ns ? kStep : 0;
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) wp[cb] += adv;
        return s >= nfull && nfull < ns ? 0 : NMAT * kChunkBytes;   // half a step at the end: its one chunk twice
    };
    i32x4 b[2][RB];
    auto read_b = [&](int stage, int kg) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) b[kg & 1][rb] = *(const i32x4 *)(lds + stage * kQ8Stage + boff[kg] + rb * 4096);
    };
    auto products = [&](int slot, int kg) {
        // a value of this place: the compiler would otherwise convert a loop-carried operand right behind its load
        uint32_t flip = 0x80808080u;
        asm volatile("" : "+s"(flip));
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) {
            const i32x4 q = signed8(w[slot][kg][cb], flip);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                acc[rb][cb] = __builtin_amdgcn_mfma_i32_32x32x32_i8(q, b[kg & 1][rb], acc[rb][cb], 0, 0, 0);
        }
    };
    // The first step's weights, then the scales and the rows, whose numbers have come meanwhile, then the other steps' weights.
    auto first_w = [&](int t) {
        const int hi = t == 0 ? NMAT * kChunkBytes : move_w(t);              // (K >= 128: the first step is whole)
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) {
            load_w(t, kg, hi);
            __builtin_amdgcn_sched_barrier(0);       // in the order in which they are used
        }
    };
    first_w(0);
    // the scales of the tile's rows and of its matrix channels, for the epilogue: one of each per thread
    float *scales = (float *)(lds + kQ8Scales);
    {
        const int ch0 = cblock * kQ8Waves * (NMAT == 2 ? 32 : 64);          // up: threads 0 .. 127, gate: 128 .. 255
        const int ch = min(ch0 + (NMAT == 2 ? tid & 127 : tid), a.NT * 16 - 1);
        const uint32_t at = lds_base + kQ8Scales + wave * 256;
        dma4(a.x_scale + row_sc, at);
        dma4((NMAT == 2 ? (tid < 128 ? slab.s_up : slab.s_gate) : slab.s_down) + ch, at + 1024);
        if (NMAT == 1) {
            if (a.bias) dma4(a.bias + ch, at + 2048);
            else scales[512 + tid] = 0.f;
        }
    }
    const uint8_t *xsrc[RB];
    // half a step at the end: lanes of its upper half re-read the lower one (q8_key of a row differs from lane >> 3 in its
    // lowest bit alone, so a lane has pieces of the same half in every row)
    const int32_t tail_fix = (((lane & 7) ^ (lane >> 3)) & 4) ? 64 : 0;
#pragma unroll
    for (int i = 0; i < RB; ++i) {
        const int piece = (lane & 7) ^ q8_key((wave * RB + i) * 8 + (lane >> 3));
        xsrc[i] = a.x + (int64_t)row[i] * a.Kdim + piece * 16;
    }
    // DMAs of step s into its stage (steps past the last one repeat it: in bounds, into a stage that is free)
    auto issue = [&](int s, int stage) {
        const int sc = min(s, ns - 1);
#pragma unroll
        for (int i = 0; i < RB; ++i)
            dma16(xsrc[i] + (int64_t)sc * 128 - (sc == nfull ? tail_fix : 0), lds_base + stage * kQ8Stage + (wave * RB + i) * 1024);
    };
#pragma unroll
    for (int t = 0; t < D; ++t) issue(t, t);
#pragma unroll
    for (int t = 1; t < D; ++t) first_w(t);
    wait_vmcnt<(D - 1) * (RB + 8)>();  // step 0's DMAs have landed: the other steps' are younger, and their weights
    block_barrier();
    read_b(0, 0);

    // Step s (slot = stage = s % 3), one k-group after the other: the rows' fragments of the next k-group are read, the
    // products of this one run, its weight registers are loaded for step s + 3.  Before the last k-group, whose
    // fragments have been read, the workgroup meets: every wave is done with this stage, which takes step s + 3,
    // and step s + 1 is in LDS, whose first fragments are read behind the last k-group's products.  In a full round a step's
    // DMAs are followed by at least RB + 16 younger loads when they are waited for: every step issues the same number of
    // loads, those for steps past the last repeat what is there (the loop carries them, so the compiler cannot drop them).
    // The one or two steps behind the last full round (REST) load nothing and wait for everything.  The fences keep the
    // compiler from gathering the loads at the end of the step, and from converting all weights at its start (which
    // would wait for the last of them).
    auto step = [&](int s, auto slot_c, auto rest_c) {
        constexpr int SLOT = decltype(slot_c)::value, NEXT = (SLOT + 1) % D;
        constexpr bool REST = decltype(rest_c)::value;
        const int hi = REST ? 0 : move_w(s + D);
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) {
            if (kg == 3) {
                wait_vmcnt<REST ? 0 : (D - 2) * (RB + 8) + 8>();
                block_barrier();
                if constexpr (!REST) issue(s + D, SLOT);
                read_b(NEXT, 0);
            } else {
                read_b(SLOT, kg + 1);
            }
            if (kg < 2 || s < nfull) products(SLOT, kg);             // half a step at the end has two k-groups
            if constexpr (!REST) load_w(SLOT, kg, hi);
            __builtin_amdgcn_sched_group_barrier(0x100, RB, 0);      // the LDS reads first
            __builtin_amdgcn_sched_group_barrier(0x008, 2 * RB, 0);
            if constexpr (!REST) __builtin_amdgcn_sched_group_barrier(0x020, 2, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // D steps a round (the loop has no other way out, so that the compiler's own waits are those of a full ring)
    auto steps = [&](auto self, int s, auto slot_c) -> void {
        constexpr int SLOT = decltype(slot_c)::value;
        step(s, slot_c, std::false_type{});
        if constexpr (SLOT + 1 < D) self(self, s + 1, std::integral_constant<int, SLOT + 1>{});
    };
    auto rest = [&](auto self, int s, auto slot_c) -> void {
        constexpr int SLOT = decltype(slot_c)::value;
        if (s >= ns) return;
        step(s, slot_c, std::true_type{});
        if constexpr (SLOT + 2 < D) self(self, s + 1, std::integral_constant<int, SLOT + 1>{});
    };
    int s = 0;
    for (; s + D <= ns; s += D) steps(steps, s, std::integral_constant<int, 0>{});
    rest(rest, s, std::integral_constant<int, 0>{});
    wait_vmcnt<0>();                  // the repeated loads

    // Epilogue.  Register 4 q + r of a lane: channel 8 q + 4 kh + r of its block, row l32 of row block rb.  The values
    // become 16-bit rows in the wave's scratch and leave in 16-byte pieces.
    uint8_t *scratch = lds + kQ8Stages * kQ8Stage + wave * kQ8Scratch;
    constexpr int NC = NMAT == 2 ? 32 : 64;                      // output channels of the wave
    const int c0 = nt0 * 16;
    const int nch = min(a.N - c0, NC);
    constexpr int PPR = NC / 8;                                  // 16-byte pieces per row
    const bool whole = nch == NC && (a.out_stride & 7) == 0;
    auto sum_of = [](int v) { return WRAP ? __builtin_elementwise_add_sat(v, 1) : v; };
    // (the lane's number asked for again: kept through the steps it was the one register too many)
    const int elane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    typedef T T4 __attribute__((ext_vector_type(4)));
    float ws[2][16], bias[2][16];
#pragma unroll
    for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float *sp = scales + 256 + (NMAT == 2 ? cb * 128 + wave * 32 : wave * 64 + cb * 32) + q * 8 + kh * 4;
            const float4 v = *(const float4 *)sp;
            ws[cb][q * 4] = v.x; ws[cb][q * 4 + 1] = v.y; ws[cb][q * 4 + 2] = v.z; ws[cb][q * 4 + 3] = v.w;
            if (NMAT == 1) {
                const float4 t = *(const float4 *)(sp + 256);
                bias[cb][q * 4] = t.x; bias[cb][q * 4 + 1] = t.y; bias[cb][q * 4 + 2] = t.z; bias[cb][q * 4 + 3] = t.w;
            }
        }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float xs = scales[rb * 32 + l32];
#pragma unroll
        for (int cb = 0; cb < (NMAT == 2 ? 1 : 2); ++cb)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = q * 4 + r;
                    v[r] = as_fp32((float)sum_of(acc[rb][cb][i]) * (xs * ws[cb][i]));
                }
                T4 o;
                if constexpr (NMAT == 2) {
                    float gate[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) gate[r] = as_fp32((float)sum_of(acc[rb][1][q * 4 + r]) * (xs * ws[1][q * 4 + r]));
                    o = swiglu4_rounded<T>(v, gate);
                } else {
                    if (a.bias) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] += bias[cb][q * 4 + r];
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = (T)v[r];
                }
                *(T4 *)(scratch + l32 * kQ8ScratchPitch + (cb * 32 + q * 8 + kh * 4) * 2) = o;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < 32 * PPR / 64; ++i) {
            const int r = (i * 64 + elane) / PPR, c = (elane % PPR) * 8;
            if (rb * 32 + r >= n) continue;
            T *orow = (T *)a.out + (int64_t)(row0 + rb * 32 + r) * a.out_stride + c0;
            const uint8_t *src = scratch + r * kQ8ScratchPitch + c * 2;
            if (whole) {
                *(uint4 *)(orow + c) = *(const uint4 *)src;
            } else {
                for (int k = 0; k < 8; ++k)
                    if (c + k < nch) orow[c + k] = ((const T *)src)[k];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// Tiles are numbered in groups of `group` items, channel block by channel block within a group; XCD x (workgroups
// x, x + 8, ...) walks a contiguous eighth of them, so that the workgroups that share an item's rows or an expert's
// weights run side by side on one L2.
template <typename T, int NMAT, bool WRAP>
__global__ __launch_bounds__(64 * kQ8Waves, 1) void q8_tile_kernel(Q8Args a, int cblocks, int group)
{
    extern __shared__ __align__(1024) uint8_t q8_lds[];
    const uint32_t items = a.dense_rows > 0 ? (uint32_t)((a.dense_rows + kQ8Rows - 1) / kQ8Rows) : (uint32_t)((ConstInts)(uintptr_t)a.lists.count)[kListT128];
    const uint32_t tiles = items * (uint32_t)cblocks, per = (tiles + 7) >> 3, at = blockIdx.x >> 3;
    const uint32_t tile = (blockIdx.x & 7) * per + at;
    if (at >= per || tile >= tiles) return;
    const uint32_t in_full = (uint32_t)group * cblocks, g = tile / in_full, rem = tile - g * in_full;
    const uint32_t in_group = min((uint32_t)group, items - g * group);
    const int cblock = (int)(rem / in_group), it = (int)(g * group + rem % in_group);
    int e = 0, row0, n;
    if (a.dense_rows > 0) {
        row0 = it * kQ8Rows;
        n = (int)min((int64_t)kQ8Rows, a.dense_rows - row0);
    } else {
        const ConstInts item = (ConstInts)(uintptr_t)(a.lists.items[kListT128] + it);
        e = item[0]; row0 = item[1]; n = item[2];
    }
    const ConstWords slab = (ConstWords)(uintptr_t)(a.slabs + e);
    switch ((n + 31) >> 5) {
    case 1: q8_tile<T, NMAT, 1, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    case 2: q8_tile<T, NMAT, 2, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    case 3: q8_tile<T, NMAT, 3, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    case 4: q8_tile<T, NMAT, 4, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    case 5: q8_tile<T, NMAT, 5, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    case 6: q8_tile<T, NMAT, 6, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    case 7: q8_tile<T, NMAT, 7, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    default: q8_tile<T, NMAT, 8, WRAP>(a, slab, row0, n, cblock, q8_lds); break;
    }
}

template <typename T, int NMAT>
static hipError_t launch_tiles(const Q8Args &a, int64_t max_items, hipStream_t s)
{
    const int per = NMAT == 2 ? 2 * kQ8Waves : 4 * kQ8Waves;    // 16-channel tiles per workgroup
    const int cblocks = (a.NT + per - 1) / per;
    const int64_t tiles = max_items * cblocks, grid = (tiles + 7) / 8 * 8;
    if (grid >= (int64_t)1 << 24) return hipErrorInvalidValue;          // threads of a launch
    const int group = a.dense_rows > 0 ? 4 : 1;
    if (a.Kdim >> 6 >= kQ8WrapChunks)
        hipLaunchKernelGGL((q8_tile_kernel<T, NMAT, true>), dim3((unsigned)grid), dim3(64 * kQ8Waves), kQ8Lds, s, a, cblocks, group);
    else
        hipLaunchKernelGGL((q8_tile_kernel<T, NMAT, false>), dim3((unsigned)grid), dim3(64 * kQ8Waves), kQ8Lds, s, a, cblocks, group);
    return hipGetLastError();
}

template <typename T, int NMAT>
static hipError_t launch_lists(const Q8Args &a, const int64_t max_items[kNumLists], bool wide, hipStream_t s)
{
    const dim3 block(64 * kQ8Slices);
    if (max_items[kListStream] > 0) {
        const unsigned items = (unsigned)max_items[kListStream];
        constexpr int NG = 4 / NMAT;
        if (wide)
            hipLaunchKernelGGL((q8_stream_kernel<T, NMAT, NG, 2, 2>), dim3((unsigned)((a.NT + NG - 1) / NG), items, kWideRows / 32), block, 0, s,
                               a, kListStream, 0);
        else
            hipLaunchKernelGGL((q8_stream_kernel<T, NMAT, 1, 1, 2>), dim3((unsigned)a.NT, items), block, 0, s, a, kListStream, 0);
    }
    if (max_items[kListT128] > 0) {
        const hipError_t e = launch_tiles<T, NMAT>(a, max_items[kListT128], s);
        if (e != hipSuccess) return e;
    }
    return hipGetLastError();
}

hipError_t launch_ffn_q8(const Q8Args &a, int stage, int act, const int64_t max_items[kNumLists], bool wide, hipStream_t s)
{
    if (act == 0)
        return stage == 1 ? launch_lists<__bf16, 2>(a, max_items, wide, s) : launch_lists<__bf16, 1>(a, max_items, wide, s);
    return stage == 1 ? launch_lists<_Float16, 2>(a, max_items, wide, s) : launch_lists<_Float16, 1>(a, max_items, wide, s);
}

template <typename T> static hipError_t launch_dense_t(const Q8Args &a, hipStream_t s)
{
    const int64_t n = a.dense_rows;
    const dim3 block(64 * kQ8Slices);
    if (n <= 16)
        hipLaunchKernelGGL((q8_stream_kernel<T, 1, 1, 1, 2>), dim3((unsigned)a.NT, 1), block, 0, s, a, 0, 16);
    else if (n <= 65535 * 32 && q8_stream_us(n, a.Kdim, a.NT * 16) < q8_tile_us(n, a.Kdim, a.NT * 16))      // (grid.y)
        hipLaunchKernelGGL((q8_stream_kernel<T, 1, 4, 2, 2>), dim3((unsigned)((a.NT + 3) / 4), (unsigned)((n + 31) / 32)), block, 0, s, a, 0, 32);
    else
        return launch_tiles<T, 1>(a, (n + kQ8Rows - 1) / kQ8Rows, s);
    return hipGetLastError();
}

hipError_t launch_dense_q8(const Q8Args &a, int act, hipStream_t s)
{
    if (a.dense_rows <= 0) return hipSuccess;
    return act == 0 ? launch_dense_t<__bf16>(a, s) : launch_dense_t<_Float16>(a, s);
}

template <typename T> static hipError_t launch_pairs_t(const Q8Args &up, const Q8Args &down, const PairArgs &pa, hipStream_t s)
{
    const int T_ = pa.P / pa.K, rows = pa.P + (pa.shared ? T_ : 0);
    hipLaunchKernelGGL(q8_pairs_up_kernel<T>, dim3((unsigned)up.NT, (unsigned)rows), dim3(64 * kQ8Slices), pa.x16 ? up.Kdim : 0, s, up, pa);
    const int waves = pa.K + (pa.shared ? 1 : 0);
    hipLaunchKernelGGL(q8_pairs_down_kernel<T>, dim3((unsigned)((down.NT + kPairTiles - 1) / kPairTiles), (unsigned)T_), dim3(64 * waves),
                       (size_t)waves * down.Kdim, s, down, pa);
    return hipGetLastError();
}

hipError_t launch_pairs_q8(const Q8Args &up, const Q8Args &down, const PairArgs &pa, int act, hipStream_t s)
{
    if (pa.P <= 0) return hipSuccess;
    if (!q8_pairs_fit(pa.P, pa.K, up.Kdim, down.Kdim)) return hipErrorInvalidValue;
    return act == 0 ? launch_pairs_t<__bf16>(up, down, pa, s) : launch_pairs_t<_Float16>(up, down, pa, s);
}

}  // namespace ek
