// attn_masked.h -- what the kernels of masked attention share: arguments, the score of a
// (row, key) pair, which keys a row sees, and one row computed by one warp.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ceb_am {

struct Args {
    const void *q, *k, *v;
    void* out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    const int32_t *cu_q, *cu_k, *prefix, *doc_q, *doc_k;
    const float *slopes, *table;
    int n_head, group, head_dim, n_seqs, q_rows, k_rows, max_q, max_k;
    int left, right, radius;  // left / right: -1 open
    float scale, cap;         // cap 0: none
    int* err;
};

// The kernels (attn_masked_f16.cu, attn_masked_bf16.cu).
int launch_f16(const Args& a, cudaStream_t st);
int launch_bf16(const Args& a, cudaStream_t st);

// One sequence: query rows q0 .. q0+n-1, key rows k0 .. k0+m-1, the first `prefix` keys seen
// by every row.
struct Seq {
    int q0, n, k0, m, prefix;
};
// False (reported if `report`) when the offsets disagree with the bounds of the call.
CEB_DEV bool load_seq(const Args& a, int s, bool report, Seq& q) {
    const int q0 = a.cu_q[s], q1 = a.cu_q[s + 1], k0 = a.cu_k[s], k1 = a.cu_k[s + 1];
    const bool ok = q0 >= 0 && q1 >= q0 && q1 <= a.q_rows && q1 - q0 <= a.max_q && k0 >= 0 && k1 >= k0 &&
                    k1 <= a.k_rows && k1 - k0 <= a.max_k;
    if (!ok) {
        if (report && a.err) atomicCAS(a.err, 0, (int)CEB_DEVERR_BAD_INDEX);
        return false;
    }
    q.q0 = q0;
    q.n = q1 - q0;
    q.k0 = k0;
    q.m = k1 - k0;
    q.prefix = a.prefix ? max(0, min(a.prefix[s], q.m)) : 0;
    return true;
}
// The window [lo, hi) of the row at place p (= i + m - n, negative for rows before the keys).
CEB_DEV void window(const Args& a, const Seq& s, int p, int& lo, int& hi) {
    lo = a.left < 0 ? 0 : (int)max((int64_t)p - a.left, (int64_t)0);
    hi = a.right < 0 ? s.m : (int)min((int64_t)p + a.right + 1, (int64_t)s.m);
    hi = max(hi, 0);
    lo = min(lo, hi);
}

CEB_DEV float bits_f(uint32_t u, __half) { return __half2float(__ushort_as_half((unsigned short)u)); }
CEB_DEV float bits_f(uint32_t u, __nv_bfloat16) { return __uint_as_float(u << 16); }
CEB_DEV float value_f(__half v) { return __half2float(v); }
CEB_DEV float value_f(__nv_bfloat16 v) { return __bfloat162float(v); }
CEB_DEV void store_f(__half* p, float v) { *p = __float2half_rn(v); }
CEB_DEV void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Row i of sequence s for one head, by one warp: a lane scores one key of 32, then every
// lane carries the head's values lane, lane + 32, ...  Only keys that the row sees are read
// into the sums, so what hidden keys hold cannot reach the result; one pass, with the
// running maximum and sum of the softmax.  It takes its time (0.2 to 0.4 us a key): `beat`, if given, is
// set to the clock all along, for waits that others bound.
template <typename T>
__device__ __noinline__ void warp_row(const Args& a, const Seq& s, int i, int head, volatile int* beat = nullptr) {
    const int lane = threadIdx.x & 31, hd = a.head_dim, kvh = head / a.group;
    const int p = i + s.m - s.n;
    int lo, hi;
    window(a, s, p, lo, hi);
    const T* q = static_cast<const T*>(a.q) + (int64_t)(s.q0 + i) * a.q_row + head * a.q_head;
    const T* kp = static_cast<const T*>(a.k) + (int64_t)s.k0 * a.k_row + kvh * a.k_head;
    const T* vp = static_cast<const T*>(a.v) + (int64_t)s.k0 * a.v_row + kvh * a.v_head;
    const int doc = a.doc_q ? a.doc_q[s.q0 + i] : 0;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    const float* table = a.table ? a.table + (int64_t)head * (2 * (int64_t)a.radius + 1) + a.radius : nullptr;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    // the keys of the prefix, then those of the window behind it
    int j0 = s.prefix > 0 ? 0 : lo / 32 * 32;
    while (j0 < max(hi, s.prefix)) {
        if (beat && lane == 0) *beat = (int)clock();
        const int j = j0 + lane;
        bool seen = j < s.m && (j < s.prefix || (j >= lo && j < hi));
        if (seen && a.doc_k) seen = doc >= 0 && a.doc_k[s.k0 + j] == doc;
        const unsigned live = __ballot_sync(0xffffffffu, seen);
        if (live) {
            float t = -INFINITY;
            if (seen) {
                const T* kr = kp + (int64_t)j * a.k_row;
                t = 0.0f;
                for (int d = 0; d < hd; d += 8) {
                    const uint4 x = *reinterpret_cast<const uint4*>(q + d), y = *reinterpret_cast<const uint4*>(kr + d);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        t = fmaf(bits_f(xs[c] & 0xffffu, T()), bits_f(ys[c] & 0xffffu, T()), t);
                        t = fmaf(bits_f(xs[c] >> 16, T()), bits_f(ys[c] >> 16, T()), t);
                    }
                }
                t *= a.scale;
                if (a.cap > 0.0f) t = a.cap * tanhf(t / a.cap);
                if (a.slopes) t -= slope * fabsf((float)(j - p));
                if (table) t += table[(int)max(-(int64_t)a.radius, min((int64_t)a.radius, (int64_t)j - p))];
            }
            float mx = t;
#pragma unroll
            for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.0f : m_new;
            const float f = expf(m - base);  // 0 for the first keys (m = -inf)
            const float w = seen ? expf(t - base) : 0.0f;
            m = m_new;
            l *= f;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= f;
            float sum = w;
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l += sum;
            for (unsigned b = live; b; b &= b - 1) {
                const int t32 = __ffs(b) - 1;
                const float wt = __shfl_sync(0xffffffffu, w, t32);
                const T* vr = vp + (int64_t)(j0 + t32) * a.v_row;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (lane + 32 * c < hd) acc[c] = fmaf(wt, value_f(vr[lane + 32 * c]), acc[c]);
            }
        }
        j0 += 32;
        if (j0 >= s.prefix && j0 < lo / 32 * 32) j0 = lo / 32 * 32;
    }
    T* o = static_cast<T*>(a.out) + (int64_t)(s.q0 + i) * a.o_row + head * a.o_head;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (lane + 32 * c < hd) store_f(o + lane + 32 * c, l == 0.0f ? 0.0f : acc[c] / l);
}

}  // namespace ceb_am
