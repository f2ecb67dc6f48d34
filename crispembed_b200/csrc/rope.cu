// rope.cu -- rotary positions as an operator: plans (frequencies, scaled for long
// contexts) and the rotation of packed rows.
//
// Pair i of a head turns by the angle p f_i, p the row's position.  Far positions need
// the product exactly: at p = 10^5 an fp32 product is off by up to 4e-3 rad.  The plan
// keeps f_i / 2 pi in 64 bits, the kernel forms the number of turns p f_i / 2 pi in 64
// bits, drops the whole turns and takes sin and cos of the rest in fp32, once per (row,
// pair) for all heads of the row.
//
// Bound by memory (70k rows x 24 heads of 64: 79.7 us, 5.4 TB/s): every value is read and written once.  A block takes some rows, puts
// their cos and sin into shared memory, then streams the rows with one 16-byte vector (two
// in the half layout: both partners) per thread and step.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "../../include/ceb_ops.h"
#include "ceb_internal.h"
#include "common.cuh"

struct ceb_rope {
    int rot_dim = 0;
    float stretch = 1.0f;     // factor of cos and sin
    int device = 0;
    double* turns = nullptr;  // [rot_dim / 2] f_i / 2 pi, on `device`
};

namespace {

constexpr int MAX_PAIRS = 128;   // rot_dim <= 256
constexpr int TABLE = 2048;      // (cos, sin) entries of a block: 16 KB
constexpr int NTHR = 256;

struct RopeArgs {
    const void* x;
    void* out;
    const double* turns;
    const int32_t* positions;
    const int32_t* cu;
    int64_t x_row, x_head, o_row, o_head;
    int n_rows, n_head, head_dim, pairs, n_seqs, pos_offset, rows_per_block;
    float stretch;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};
CEB_DEV float to_f(float v) { return v; }
CEB_DEV float to_f(__half v) { return __half2float(v); }
CEB_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
CEB_DEV void from_f(float v, float& o) { o = v; }
CEB_DEV void from_f(float v, __half& o) { o = __float2half_rn(v); }
CEB_DEV void from_f(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }

// The last s of 0 .. n with cu[s] <= row (-1: none), by a whole warp: 32 probes a step.
CEB_DEV int warp_find(const int32_t* __restrict__ cu, int n, int row, int lane) {
    int lo = -1, hi = n + 1;  // cu[lo] <= row < cu[hi]
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = lo + 1 + lane * step;
        const unsigned le = __ballot_sync(0xffffffffu, at < hi && cu[at] <= row);
        const int k = le ? 31 - __clz(le) : -1;  // the highest probe not past the row
        const int l = k < 0 ? lo : lo + 1 + k * step;
        hi = min(hi, k < 0 ? lo + 1 : l + step);
        lo = l;
    }
    return lo;
}

// V: values a vector; half layout: the unit holds V pairs (two vectors, rot_dim/2 apart);
// interleaved: V/2 pairs (one vector; V = 1: one pair as two single values).
template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(NTHR) rope_kernel(const RopeArgs a) {
    __shared__ float2 cs[TABLE];
    __shared__ int64_t pos[NTHR / 32 * 2];
    const int tid = threadIdx.y * blockDim.x + threadIdx.x, n_thr = blockDim.x * blockDim.y;
    const int row0 = blockIdx.x * a.rows_per_block;
    const int rows = min(a.rows_per_block, a.n_rows - row0);
    const int warp = tid >> 5, lane = tid & 31, n_warps = n_thr >> 5;
    for (int r = warp; r < rows; r += n_warps) {
        int64_t p;
        if (a.positions) {
            p = a.positions[row0 + r];
        } else {
            const int s = warp_find(a.cu, a.n_seqs, row0 + r, lane);
            p = s < 0 || s >= a.n_seqs ? INT64_MIN : (int64_t)(row0 + r) - a.cu[s] + a.pos_offset;
        }
        if (lane == 0) pos[r] = p;
    }
    __syncthreads();
    for (int i = tid; i < rows * a.pairs; i += n_thr) {
        const int r = i / a.pairs, j = i - r * a.pairs;
        const double t = (double)pos[r] * a.turns[j];
        float sn, c;
        sincospif(2.0f * (float)(t - rint(t)), &sn, &c);
        cs[i] = make_float2(c * a.stretch, sn * a.stretch);
    }
    __syncthreads();
    constexpr bool SINGLE = INTER && V == 1;
    // Rows whose loads go out before the first is needed: four vectors a thread (two rows of two in the
    // half layout).  95k rows x 10 heads of 128, half of each interleaved: one row at a time 96 us, four
    // 88, eight 119 (registers).  70k rows x 24 heads of 64, half layout: two rows 79.7, four 82.
    constexpr int DEEP = INTER ? 4 : 2;
    constexpr int P = INTER && !SINGLE ? V / 2 : V;  // pairs a unit
    const int units = a.pairs / P;        // per head
    const int total = a.n_head * units;
    const bool copy = a.x != a.out;
    const int tail = copy ? (a.head_dim - 2 * a.pairs) / V : 0;  // vectors behind the rotated values
    for (int e = threadIdx.x; e < total; e += blockDim.x) {
        const int h = e / units, u = e - h * units;
        const int at = SINGLE ? 2 * u : u * V;
        const T* x = static_cast<const T*>(a.x) + (int64_t)row0 * a.x_row + h * a.x_head + at;
        T* o = static_cast<T*>(a.out) + (int64_t)row0 * a.o_row + h * a.o_head + at;
        for (int r0 = threadIdx.y; r0 < rows; r0 += DEEP * blockDim.y) {
            if constexpr (SINGLE) {
#pragma unroll
                for (int d = 0; d < DEEP; ++d) {
                    const int r = r0 + d * blockDim.y;
                    if (r >= rows || pos[r] == INT64_MIN) continue;
                    const float x0 = to_f(x[r * a.x_row]), x1 = to_f(x[r * a.x_row + 1]);
                    const float2 t = cs[r * a.pairs + u];
                    from_f(x0 * t.x - x1 * t.y, o[r * a.o_row]);
                    from_f(x0 * t.y + x1 * t.x, o[r * a.o_row + 1]);
                }
            } else {
                Vec<T, V> p[DEEP], q[INTER ? 1 : DEEP];
                bool on[DEEP];
#pragma unroll
                for (int d = 0; d < DEEP; ++d) {
                    const int r = r0 + d * blockDim.y;
                    on[d] = r < rows && pos[r] != INT64_MIN;
                    if (on[d]) {
                        p[d] = *reinterpret_cast<const Vec<T, V>*>(x + r * a.x_row);
                        if constexpr (!INTER) q[d] = *reinterpret_cast<const Vec<T, V>*>(x + r * a.x_row + a.pairs);
                    }
                }
#pragma unroll
                for (int d = 0; d < DEEP; ++d) {
                    if (!on[d]) continue;
                    const int r = r0 + d * blockDim.y;
                    const float2* w = cs + r * a.pairs + u * P;
                    Vec<T, V> y;
                    if constexpr (INTER) {
#pragma unroll
                        for (int j = 0; j < P; ++j) {
                            const float2 t = w[j];
                            const float x0 = to_f(p[d].e[2 * j]), x1 = to_f(p[d].e[2 * j + 1]);
                            from_f(x0 * t.x - x1 * t.y, y.e[2 * j]);
                            from_f(x0 * t.y + x1 * t.x, y.e[2 * j + 1]);
                        }
                    } else {
                        Vec<T, V> z;
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float2 t = w[j];
                            const float x0 = to_f(p[d].e[j]), x1 = to_f(q[d].e[j]);
                            from_f(x0 * t.x - x1 * t.y, y.e[j]);
                            from_f(x0 * t.y + x1 * t.x, z.e[j]);
                        }
                        *reinterpret_cast<Vec<T, V>*>(o + r * a.o_row + a.pairs) = z;
                    }
                    *reinterpret_cast<Vec<T, V>*>(o + r * a.o_row) = y;
                }
            }
        }
    }
    for (int e = threadIdx.x; e < a.n_head * tail; e += blockDim.x) {
        const int h = e / tail, at = 2 * a.pairs + (e - h * tail) * V;
        const T* x = static_cast<const T*>(a.x) + (int64_t)row0 * a.x_row + h * a.x_head + at;
        T* o = static_cast<T*>(a.out) + (int64_t)row0 * a.o_row + h * a.o_head + at;
        for (int r0 = threadIdx.y; r0 < rows; r0 += DEEP * blockDim.y) {
            Vec<T, V> p[DEEP];
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const int r = r0 + d * blockDim.y;
                if (r < rows && pos[r] != INT64_MIN) p[d] = *reinterpret_cast<const Vec<T, V>*>(x + r * a.x_row);
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const int r = r0 + d * blockDim.y;
                if (r < rows && pos[r] != INT64_MIN) *reinterpret_cast<Vec<T, V>*>(o + r * a.o_row) = p[d];
            }
        }
    }
}

template <typename T, int V, bool INTER>
int launch(RopeArgs a, cudaStream_t st) {
    const int total = a.n_head * (a.pairs / (INTER && V > 1 ? V / 2 : V));
    // x: units of a row, y: rows; whole warps, since the position search is a warp's work
    int x = std::min(total, NTHR), y = NTHR / x, step = 32;
    while (step > 1 && x * (step / 2) % 32 == 0) step /= 2;
    y = y / step * step;
    if (y == 0) {
        x = (x + 31) / 32 * 32;
        y = NTHR / x;
    }
    const dim3 block(x, y);
    // few rows are spread over all SMs, many are taken up to 16 at a time
    const int cap = std::min(TABLE / a.pairs, 16);
    a.rows_per_block = std::max(1, std::min(cap, a.n_rows / (4 * ceb_num_sms())));
    const int grid = (a.n_rows + a.rows_per_block - 1) / a.rows_per_block;
    const double bytes = 2.0 * a.n_rows * a.n_head * (a.x == a.out ? 2 * a.pairs : a.head_dim) * sizeof(T);
    CEB_LAUNCH(CEB_PROF_ROWWISE, st, 0.0, bytes, rope_kernel<T, V, INTER><<<grid, block, 0, st>>>(a));
    CEB_CUDA_OK(cudaGetLastError());
    return 0;
}

// The widest vector that pointers, strides and the head's parts allow.
template <typename T>
int dispatch(const RopeArgs& a, bool inter, cudaStream_t st) {
    auto fits = [&](int v) {
        const int64_t strides = a.x_row | a.x_head | a.o_row | a.o_head | a.head_dim | (inter ? 2 * a.pairs : a.pairs);
        const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out);
        return strides % v == 0 && ptrs % (v * sizeof(T)) == 0;
    };
    constexpr int W = 16 / sizeof(T);
    if (inter) {
        if (fits(W)) return launch<T, W, true>(a, st);
        if (fits(2)) return launch<T, 2, true>(a, st);
        return launch<T, 1, true>(a, st);
    }
    if (fits(W)) return launch<T, W, false>(a, st);
    if (fits(2)) return launch<T, 2, false>(a, st);
    return launch<T, 1, false>(a, st);
}

}  // namespace

extern "C" ceb_rope* ceb_rope_create(int rot_dim, double theta, int scaling, double factor, int context,
                                     double beta_fast, double beta_slow) {
    auto bad = [](const char* why) {
        ceb_set_error(1, "rope_create: %s", why);
        return static_cast<ceb_rope*>(nullptr);
    };
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 2 * MAX_PAIRS) return bad("rot_dim must be even, 2 to 256");
    if (!(theta > 1.0) || !std::isfinite(theta)) return bad("theta must be a finite number above 1");
    if (scaling < CEB_ROPE_NONE || scaling > CEB_ROPE_YARN) return bad("unknown scaling");
    if (!(factor >= 1.0) || !std::isfinite(factor)) return bad("factor must be a finite number of at least 1");
    if (scaling == CEB_ROPE_NTK && rot_dim == 2) return bad("NTK scaling needs rot_dim above 2");
    if (scaling == CEB_ROPE_YARN &&
        (context <= 0 || !(beta_slow > 0.0) || !(beta_fast > beta_slow) || !std::isfinite(beta_fast)))
        return bad("YARN scaling needs context > 0 and beta_fast > beta_slow > 0");
    const int n = rot_dim / 2;
    const double pi = 3.14159265358979323846;
    double turns[MAX_PAIRS];
    if (scaling == CEB_ROPE_NTK) theta *= std::pow(factor, rot_dim / (rot_dim - 2.0));
    double low = 0.0, high = 0.0;
    if (scaling == CEB_ROPE_YARN) {
        // pair i turns context * f_i / 2 pi times; solved for i at beta turns
        auto pair_of = [&](double beta) {
            return rot_dim * std::log(context / (beta * 2.0 * pi)) / (2.0 * std::log(theta));
        };
        low = std::max(std::floor(pair_of(beta_fast)), 0.0);
        high = std::min(std::ceil(pair_of(beta_slow)), rot_dim - 1.0);
    }
    for (int i = 0; i < n; ++i) {
        double f = std::pow(theta, -2.0 * i / rot_dim);
        if (scaling == CEB_ROPE_LINEAR) f /= factor;
        if (scaling == CEB_ROPE_YARN) {
            const double g = std::min(std::max((i - low) / std::max(high - low, 1e-3), 0.0), 1.0);
            f = f / factor * g + f * (1.0 - g);
        }
        turns[i] = f / (2.0 * pi);
    }
    ceb_rope* R = new (std::nothrow) ceb_rope;
    if (!R) return bad("out of host memory");
    R->rot_dim = rot_dim;
    R->stretch = scaling == CEB_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    cudaError_t e = cudaGetDevice(&R->device);
    if (e == cudaSuccess) e = cudaMalloc(&R->turns, n * sizeof(double));
    // On a stream of its own that is waited for: a copy on the legacy stream may return before it has
    // landed, and streams that do not wait for that one could read the plan too early.
    cudaStream_t own = nullptr;
    if (e == cudaSuccess) e = cudaStreamCreateWithFlags(&own, cudaStreamNonBlocking);
    if (e == cudaSuccess) e = cudaMemcpyAsync(R->turns, turns, n * sizeof(double), cudaMemcpyHostToDevice, own);
    if (e == cudaSuccess) e = cudaStreamSynchronize(own);
    if (own) cudaStreamDestroy(own);
    if (e != cudaSuccess) {
        cudaGetLastError();
        ceb_set_cuda_error(e, "rope_create", __FILE__, __LINE__);
        ceb_rope_free(R);
        return nullptr;
    }
    return R;
}

extern "C" void ceb_rope_free(ceb_rope* R) {
    if (!R) return;
    if (R->turns) cudaFree(R->turns);
    delete R;
}

extern "C" int ceb_rope_forward(const ceb_rope* R, const void* d_x, void* d_out, int dtype, int n_rows, int n_head,
                                int head_dim, int64_t x_row, int64_t x_head, int64_t o_row, int64_t o_head,
                                int interleaved, const int32_t* d_positions, const int32_t* d_cu_seqlens, int n_seqs,
                                int pos_offset, void* stream) {
    if (!R || n_rows < 0 || n_head <= 0 || n_seqs < 0) return ceb_set_error(1, "rope: bad arguments");
    if (dtype != CEB_ACT_F32 && dtype != CEB_ACT_BF16 && dtype != CEB_ACT_F16)
        return ceb_set_error(1, "rope: dtype %d unsupported", dtype);
    if (head_dim < R->rot_dim) return ceb_set_error(1, "rope: head_dim %d below rot_dim %d", head_dim, R->rot_dim);
    if (n_rows == 0) return 0;
    if (!d_x || !d_out) return ceb_set_error(1, "rope: null tensor");
    if (!d_positions && (!d_cu_seqlens || n_seqs == 0))
        return ceb_set_error(1, "rope: positions or cu_seqlens must be given");
    const int esz = dtype == CEB_ACT_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_out)) % esz)
        return ceb_set_error(1, "rope: tensors must be aligned to their type");
    if (n_head == 1) x_head = o_head = 0;
    // the heads of a row, or the rows of a head, lie apart
    auto apart = [&](int64_t row, int64_t head) {
        const int64_t in_row = (n_head - 1) * head + head_dim, in_head = (n_rows - 1) * row + head_dim;
        if (row < 0 || head < 0 || (n_head > 1 && head < head_dim) || (n_rows > 1 && row < head_dim)) return false;
        return n_rows == 1 || row >= in_row || (n_head == 1 || head >= in_head);
    };
    if (!apart(x_row, x_head) || !apart(o_row, o_head))
        return ceb_set_error(1, "rope: strides must keep rows and heads of %d values apart", head_dim);
    const int64_t span_x = ((n_rows - 1) * x_row + (n_head - 1) * x_head + head_dim) * esz;
    const int64_t span_o = ((n_rows - 1) * o_row + (n_head - 1) * o_head + head_dim) * esz;
    const uint8_t *px = static_cast<const uint8_t*>(d_x), *po = static_cast<const uint8_t*>(d_out);
    const bool same = px == po && (n_rows == 1 || x_row == o_row) && x_head == o_head;
    if (!same && px < po + span_o && po < px + span_x)
        return ceb_set_error(1, "rope: out overlaps x without being x");
    int dev = -1;
    CEB_CUDA_OK(cudaGetDevice(&dev));
    if (dev != R->device)
        return ceb_set_error(1, "rope: plan of device %d used on device %d", R->device, dev);
    RopeArgs a;
    a.x = d_x;
    a.out = d_out;
    a.turns = R->turns;
    a.positions = d_positions;
    a.cu = d_cu_seqlens;
    a.x_row = n_rows == 1 ? 0 : x_row;
    a.o_row = n_rows == 1 ? 0 : o_row;
    a.x_head = x_head;
    a.o_head = o_head;
    a.n_rows = n_rows;
    a.n_head = n_head;
    a.head_dim = head_dim;
    a.pairs = R->rot_dim / 2;
    a.n_seqs = n_seqs;
    a.pos_offset = pos_offset;
    a.stretch = R->stretch;
    a.rows_per_block = 1;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool inter = interleaved != 0;
    return dtype == CEB_ACT_F32   ? dispatch<float>(a, inter, st)
           : dtype == CEB_ACT_F16 ? dispatch<__half>(a, inter, st)
                                  : dispatch<__nv_bfloat16>(a, inter, st);
}
