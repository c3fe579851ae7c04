// Products of int8 activation rows with int8 weights: the two stages of the expert FFN on 8-bit
// activations, and one matrix alone (ek_linear).
//
//   u[n, c] = sum_k q[n, k] w[c, k] * scale[n] * w_scale[c]
//
// with the integer sum exact in int32 (|sum| <= 127 * 127 * 131072 < 2^31).  Integer addition is
// associative, so every split of the contraction and every tile shape below gives the same bits.
// Weights lie in HBM as for W8A16 (ek_internal.h): one 1 KiB chunk is the A operand of
// v_mfma_i32_16x16x64_i8 as it is, but for the offset-binary storage: q = u ^ 0x80.
#include "ek_internal.h"
#include "ek_mfma.h"

namespace ek {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i32x4 signed8(uint4 u)
{
    return i32x4{(int)(u.x ^ 0x80808080u), (int)(u.y ^ 0x80808080u), (int)(u.z ^ 0x80808080u), (int)(u.w ^ 0x80808080u)};
}

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

template <typename T, int NMAT>
static hipError_t launch_lists(const Q8Args &a, const int64_t max_items[kNumLists], bool wide, hipStream_t s)
{
    const dim3 block(64 * kQ8Slices);
    auto grid = [&](int64_t items, int parts) { return dim3((unsigned)a.NT, (unsigned)items, (unsigned)parts); };
    if (max_items[kListStream] > 0) {
        if (wide) hipLaunchKernelGGL((q8_stream_kernel<T, NMAT, 1, 4, 2>), grid(max_items[kListStream], 1), block, 0, s, a, kListStream, 0);
        else hipLaunchKernelGGL((q8_stream_kernel<T, NMAT, 1, 1, 2>), grid(max_items[kListStream], 1), block, 0, s, a, kListStream, 0);
    }
    if (max_items[kListT32] > 0)
        hipLaunchKernelGGL((q8_stream_kernel<T, NMAT, 1, 2, 2>), grid(max_items[kListT32], 1), block, 0, s, a, kListT32, 0);
    if (max_items[kListT64] > 0)
        hipLaunchKernelGGL((q8_stream_kernel<T, NMAT, 1, 4, 2>), grid(max_items[kListT64], 1), block, 0, s, a, kListT64, 0);
    if (max_items[kListT128] > 0)
        hipLaunchKernelGGL((q8_stream_kernel<T, NMAT, 1, 4, 2>), grid(max_items[kListT128], 2), block, 0, s, a, kListT128, 0);
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
    if (n <= 16) hipLaunchKernelGGL((q8_stream_kernel<T, 1, 1, 1, 2>), dim3((unsigned)a.NT, 1), block, 0, s, a, 0, 16);
    else hipLaunchKernelGGL((q8_stream_kernel<T, 1, 1, 4, 2>), dim3((unsigned)a.NT, (unsigned)((n + 63) / 64)), block, 0, s, a, 0, 64);
    return hipGetLastError();
}

hipError_t launch_dense_q8(const Q8Args &a, int act, hipStream_t s)
{
    if (a.dense_rows <= 0) return hipSuccess;
    return act == 0 ? launch_dense_t<__bf16>(a, s) : launch_dense_t<_Float16>(a, s);
}

}  // namespace ek
