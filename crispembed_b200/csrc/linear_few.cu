// linear_few.cu -- the fused linear layer for a few rows (single tokens).
//
// A tile of the tcgen05 kernels computes 128 or 256 rows whatever the number it was given, on
// as many block pairs as the layer has 256-wide column tiles (three at 768): with few rows the
// time is the latency of that chain, 13.5 us at 768 x 768 (here: 2.8 us).  Here the weights are spread over
// the SMs and each is read once: a block takes 16 rows of W, its warps every WARPS-th block
// along k; m16n8k16 products (16 features x 8 rows of x) add up in fp32 registers, the warps'
// sums meet in shared memory in warp order, and the epilogue follows.
//
// A product's 16 k values may be any 16 as long as both operands agree: a lane takes 16 bytes
// of a weight row and the same values of a row of x as they lie in memory and feeds them to
// the products pair by pair, without a shuffle.  Quantized weights are rounded to fp16 in
// registers, as the tcgen05 kernels round them.
//
// Bound by the weights' bytes, at small layers by the latency of a launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/ceb_ops.h"
#include "ceb_internal.h"
#include "common.cuh"
#include "epilogue.cuh"

namespace {
using namespace ceb_epi;

#ifndef FEW_WARPS
#define FEW_WARPS 8
#endif
constexpr int WARPS = FEW_WARPS;
constexpr int ROWS = 16;  // of W, a block

// The 16 of a block row's 64 values that lane part t (0..3) takes, as two groups of eight
// (four fp16 pairs each) that begin at k value k(t, s).
template <int FMT>
struct Piece;
template <>
struct Piece<CEB_W_F16> {
    uint4 u[2];
    CEB_DEV void load(const uint8_t* blk, int r, int t) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
            u[s] = __ldg(reinterpret_cast<const uint4*>(blk + r * 128 + 16 * ((t + 4 * s) ^ (r & 7))));
    }
    static CEB_DEV int k(int t, int s) { return 8 * (t + 4 * s); }
    CEB_DEV void pairs(int s, uint32_t (&o)[4]) const { o[0] = u[s].x, o[1] = u[s].y, o[2] = u[s].z, o[3] = u[s].w; }
};
template <>
struct Piece<CEB_W_Q8_0> {
    uint4 u;
    uint32_t sc;  // scale of the 32-value block, fp16
    CEB_DEV void load(const uint8_t* blk, int r, int t) {
        u = __ldg(reinterpret_cast<const uint4*>(blk + r * 64 + 16 * (t ^ ((r >> 1) & 3))));
        sc = __ldg(reinterpret_cast<const unsigned short*>(blk + 8192 + 4 * r + 2 * (t >> 1)));
    }
    static CEB_DEV int k(int t, int s) { return 16 * t + 8 * s; }
    CEB_DEV void pairs(int s, uint32_t (&o)[4]) const {
        const __half2 d = __half2half2(__ushort_as_half((unsigned short)sc));
        i8x4_to_h2x2(s ? u.z : u.x, d, o[0], o[1]);
        i8x4_to_h2x2(s ? u.w : u.y, d, o[2], o[3]);
    }
};
template <>
struct Piece<CEB_W_Q4_K> {
    uint2 u;   // low nibbles: eight values, high nibbles: those 32 further
    float2 d[2];  // (scale, minimum) of the two sub-blocks
    CEB_DEV void load(const uint8_t* blk, int r, int t) {
        u = __ldg(reinterpret_cast<const uint2*>(blk + r * 32 + 16 * ((t >> 1) ^ ((r >> 2) & 1)) + 8 * (t & 1)));
        const float4 f = __ldg(reinterpret_cast<const float4*>(blk + 4096 + 16 * r));
        d[0] = make_float2(f.x, f.y);
        d[1] = make_float2(f.z, f.w);
    }
    static CEB_DEV int k(int t, int s) { return 8 * t + 32 * s; }
    CEB_DEV void pairs(int s, uint32_t (&o)[4]) const {
        const float2 f = d[s];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = ((i < 2 ? u.x : u.y) >> (4 * s)) & 0x0F0F0F0Fu;
            const int b = 2 * (i & 1);
            o[i] = h2_as_u32(__floats2half2_rn(__fsub_rn(__fmul_rn(f.x, nib_f(w, b)), f.y),
                                               __fsub_rn(__fmul_rn(f.x, nib_f(w, b + 1)), f.y)));
        }
    }
};

CEB_DEV void mma_16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: groups of eight rows of x that a block takes at most
template <int FMT, int NT>
__global__ void __launch_bounds__(32 * WARPS)
    linear_few_kernel(const uint8_t* __restrict__ q, int64_t blk_bytes, int nkb, const __half* __restrict__ x,
                      const ceb_gemm_args a) {
    using P = Piece<FMT>;
    constexpr int UNROLL = 3;
    __shared__ float red[WARPS][8 * NT][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * ROWS, m0 = blockIdx.y * 8 * NT, m = min(8 * NT, a.m_rows - m0);
    const int r = n0 % 128 + g;
    const uint8_t* blk = q + (int64_t)(n0 / 128) * nkb * blk_bytes;
    const __half* xr = x + (int64_t)(m0 + g) * a.ldx;  // rows past m are not read
    float acc[NT][4] = {};
    for (int kb0 = warp; kb0 < nkb; kb0 += WARPS * UNROLL) {
        P lo[UNROLL], hi[UNROLL];
#pragma unroll
        for (int j = 0; j < UNROLL; ++j)
            if (kb0 + WARPS * j < nkb) {
                lo[j].load(blk + (kb0 + WARPS * j) * blk_bytes, r, t);
                hi[j].load(blk + (kb0 + WARPS * j) * blk_bytes, r + 8, t);
            }
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
            const int kb = kb0 + WARPS * j;
            if (kb >= nkb) break;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t w[4], v[4];
                lo[j].pairs(s, w);
                hi[j].pairs(s, v);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    uint4 b = make_uint4(0, 0, 0, 0);
                    if (8 * i + g < m)
                        b = __ldg(reinterpret_cast<const uint4*>(xr + (int64_t)(8 * i) * a.ldx + 64 * kb + P::k(t, s)));
                    mma_16n8k16(acc[i], w[0], v[0], w[1], v[1], b.x, b.y);
                    mma_16n8k16(acc[i], w[2], v[2], w[3], v[3], b.z, b.w);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][8 * i + 2 * t + (e & 1)][g + 8 * (e >> 1)] = acc[i][e];
    __syncthreads();
    for (int e = threadIdx.x; e < m * ROWS; e += 32 * WARPS) {
        const int i = e / ROWS, n = n0 + e % ROWS;
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) y += red[w][i][e % ROWS];
        if (a.epi & CEB_EPI_BIAS) y += a.bias[n];
        y = ex_act_one(y, a.act);
        if (a.res) y += load1(a.res, a.res_type, (m0 + i) * a.ldr + n);
        store1(a.out, a.out_type, (m0 + i) * a.ldo + n, y);
    }
}

template <int FMT, int NT>
int launch(const ceb_wplane& w, const void* x, const ceb_gemm_args& a, cudaStream_t st) {
    const dim3 grid(w.n_out / ROWS, (a.m_rows + 8 * NT - 1) / (8 * NT));
    linear_few_kernel<FMT, NT><<<grid, 32 * WARPS, 0, st>>>(w.q, w.blk_bytes, w.k / 64, static_cast<const __half*>(x), a);
    CEB_CUDA_OK(cudaGetLastError());
    return 0;
}
template <int FMT>
int by_rows(const ceb_wplane& w, const void* x, const ceb_gemm_args& a, cudaStream_t st) {
    return a.m_rows <= 8 ? launch<FMT, 1>(w, x, a, st) : a.m_rows <= 16 ? launch<FMT, 2>(w, x, a, st) : launch<FMT, 4>(w, x, a, st);
}

}  // namespace

// Blocks take up to 32 rows and run two to an SM; a wave of them takes 5.2 us at k = 768 (7.7 us
// at 1536), two waves 10.1 (13.5) and three 14.6 (19.7), where the tcgen05 kernel takes 14.1 (18.0)
// for any of these sizes: two waves are the limit.  Up to eight rows a block reads little more
// than its weights, and the bytes count whatever the width.
bool ceb_linear_is_few(const ceb_wplane& w, int m) {
    return m <= 8 || (int64_t)(w.n_out / ROWS) * ((m + 31) / 32) <= 4 * ceb_num_sms();
}

int ceb_linear_few(const ceb_wplane& w, const void* x_f16, const ceb_gemm_args& a, cudaStream_t st) {
    const double flops = 2.0 * a.m_rows * w.n_out * w.k, bytes = (double)w.q_bytes + 2.0 * a.m_rows * w.k;
    int rc = 0;
    CEB_LAUNCH(a.prof_cat, st, flops, bytes,
               rc = w.format == CEB_W_F16    ? by_rows<CEB_W_F16>(w, x_f16, a, st)
                    : w.format == CEB_W_Q8_0 ? by_rows<CEB_W_Q8_0>(w, x_f16, a, st)
                                             : by_rows<CEB_W_Q4_K>(w, x_f16, a, st));
    return rc;
}
