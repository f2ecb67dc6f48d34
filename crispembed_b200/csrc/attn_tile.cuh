// attn_tile.cuh -- attention with shared key heads, score capping, a bias by distance and
// masks, over packed sequences (ceb_attention_masked), on single-CTA tcgen05 MMAs.
//
// An item is (sequence, key head, query tile).  A tile's 128 MMA rows are query rows times
// the query heads that share the key head (row r: query r / group, head r % group), so a
// key tile is read once for all of them.  Keys stream in chunks; per chunk
//   S = Q K^T   M = 128, N = the chunk's keys, fp32 in TMEM; head dims that are no multiple
//               of 64 are filled up with zeros by the loads,
//   softmax     one thread per row: score cap, bias, mask, the running maximum and sum in
//               fp32, exponentials in fp32, weights rounded to the inputs' type (the MMA's
//               operands have one type) into TMEM,
//   O += P V    P from TMEM, V MN-major from shared memory, fp32 in TMEM.
// The maximum that the exponentials use is raised -- and O rescaled -- only when the true one
// exceeds it by 2^RAISE; fp16 weights carry a factor 2^UP so that small ones stay normal
// numbers (both sums carry it, and the division drops it).
//
// A block goes on to items of blocks that have not started (cluster launch control), so
// ragged items spread over the SMs without a counter in memory: calls hold no state.  The
// loading warp runs ahead: it decodes items into a ring in shared memory, skips chunks that
// no row of the tile sees (window, prefix, document ranges) and marks chunks that need a
// mask.
//
// What hidden keys hold must not reach a sum.  Their scores are replaced before the softmax.
// In P V, 0 times inf or NaN would be NaN: rows of a V tile past the sequence's end are
// cleared, and a row whose result is not finite is computed again by one warp that reads
// visible keys only (warp_row).
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/ceb_ops.h"
#include "attn_masked.h"
#include "ceb_internal.h"

namespace {
using namespace ceb_am;

constexpr int QT = 128;   // rows of a tile (MMA M)
constexpr int NTHR = 256; // warp 0 loads, warp 1 TMEM + MMA, warps 4..7 softmax
constexpr int NRING = 4;  // items handed from the loading warp to the others

// HD: values of a head (filled up to 64 or 128); KC: keys a chunk, 64, or 96 for HD 64
template <int HD, int KC_>
struct Cfg {
    static constexpr int KC = KC_;
    static constexpr int QB = HD == 64 ? 2 : 1;             // Q buffers
    static constexpr int NS = HD == 128 ? 2 : KC == 96 ? 3 : 4;  // stages of K and of V
    static constexpr int ND = NS + 2;                       // chunk descriptions
    static constexpr int Q_BYTES = QT * HD * 2;             // 64-wide parts, one behind the other
    static constexpr int K_BYTES = KC * HD * 2;             // K or V of a chunk
    // two buffers of S, whose columns then hold P; O behind them
    static constexpr uint32_t O_COL = 2 * KC, TMEM_COLS = 256;
    static_assert(O_COL + HD <= TMEM_COLS, "TMEM plan");
    enum { B_QFULL, B_QFREE = B_QFULL + 2, B_KFULL = B_QFREE + 2, B_KFREE = B_KFULL + NS, B_VFULL = B_KFREE + NS,
           B_VFREE = B_VFULL + NS, B_SFULL = B_VFREE + NS, B_PFULL = B_SFULL + 2,
           B_PVDONE = B_PFULL + 2, B_DRAIN = B_PVDONE + 2, B_NEXT, B_IFULL, B_IFREE = B_IFULL + NRING, NBAR = B_IFREE + NRING };
};

// A decoded item: query rows i0 .. of the tile (local), its sequence, key head; `empty`: no
// key is seen by any row.  kvh < 0 ends the stream.
struct Item {
    Seq s;
    int i0, kvh, empty;
};
struct alignas(16) Chunk {
    // first key (local); 16-key steps that hold a key; slot of the documents (ONE_DOC: the document)
    int k0, flags, steps, docs;
};
constexpr int MAX_BARS = 48, MAX_ND = 6, RANGES = 256;
enum { LAST = 1, MASKED = 2, DOCS = 4, TAIL = 8, ONE_DOC = 16 };  // TAIL: the sequence ends in it

struct Small {  // shared memory behind the tiles
    uint64_t bars[MAX_BARS];
    alignas(16) uint32_t answer[4];
    uint32_t tmem;
    int abort[2];  // a role gave up; the clock when a row was last seen being computed again
    Item ring[NRING];
    Chunk chunk[MAX_ND];  // from the loading warp to the MMA warp
    Chunk now[2];         // of the S buffers, from there to the softmax
    int docs[MAX_ND][96];
    int2 range[RANGES];       // documents (least, greatest) of chunks of the sequence at hand ...
    int range_tag[RANGES / 8];  // ... of which eight each; a greatest below 0: -1 - it, a key of none is among them
    float2 ml[QT];  // (maximum, sum) of a row, for the join of a split item
};
// two warpgroups: their shares add up to the launch's 256 x 128 registers
constexpr int CONTROL_REGS = 64, ROW_REGS = 192;
static_assert(128 * (CONTROL_REGS + ROW_REGS) == NTHR * 128, "register shares");
template <int N>
CEB_DEV void regs_down() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
CEB_DEV void regs_up() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <class C>
constexpr size_t smem_bytes() {
    static_assert(C::NBAR <= MAX_BARS && C::ND <= MAX_ND, "shared memory plan");
    return 1024 + C::QB * C::Q_BYTES + 2 * C::NS * C::K_BYTES + sizeof(Small);
}
constexpr size_t two_blocks(size_t smem) { return 2 * (smem + 1024); }
static_assert(two_blocks(smem_bytes<Cfg<64, 64>>()) <= 228 * 1024 && two_blocks(smem_bytes<Cfg<64, 96>>()) <= 228 * 1024 &&
                  two_blocks(smem_bytes<Cfg<128, 64>>()) <= 228 * 1024,
              "two blocks per SM");

constexpr float LOG2E = 1.4426950408889634f;
template <typename T>
constexpr float RAISE = std::is_same<T, __half>::value ? 4.0f : 8.0f;
template <typename T>
constexpr float UP = std::is_same<T, __half>::value ? 8.0f : 0.0f;

CEB_DEV float ex2f(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
CEB_DEV float rcpf(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// c tanh(s / c) of the score s = x scale, y = s / c = x in.
// NEAR, for |y| <= 1: s P(y^2), with P fitted to tanh(y) / y on [0, 1] for least relative error (2e-7 in
//   fp32): multiply-adds alone, as good at any cap.
// FAR: c (1 - 2 / (1 + e^2y)), two special-function results a score, right to 2^-22 of c.  Up to a cap
//   of SMALL_CAP that is 2^-16 at most, a sixteenth of what rounding to fp16 does to a weight, and good
//   for any score; at a cap of 10^6 a small score would be off by 0.07.
// EACH: either one by the score's own y.
// Scores and cap may be in any units (scale2, cap2: log2).
enum { NEAR, FAR, EACH };
constexpr float SMALL_CAP = 64.0f;
template <int FORM, int N>
CEB_DEV void capped(float* x, float in, float scale2, float cap2) {
#pragma unroll
    for (int t = 0; t < N; t += 2) {
        const f32x2 x2 = f2_pack(x[t], x[t + 1]), y = f2_mul(x2, f2_splat(in)), z = f2_mul(y, y);
        if constexpr (FORM != FAR) {
            f32x2 p = f2_splat(0.0010410225950181484f);
            p = f2_fma(p, z, f2_splat(-0.0062033794820308685f));
            p = f2_fma(p, z, f2_splat(0.020289981737732887f));
            p = f2_fma(p, z, f2_splat(-0.05345702916383743f));
            p = f2_fma(p, z, f2_splat(0.13325203955173492f));
            p = f2_fma(p, z, f2_splat(-0.33332839608192444f));
            p = f2_fma(p, z, f2_splat(0.9999999403953552f));
            f2_unpack(f2_mul(f2_mul(x2, f2_splat(scale2)), p), x[t], x[t + 1]);
        }
        if constexpr (FORM != NEAR) {
            float y0, y1, e0, e1;
            f2_unpack(y, y0, y1);
            f2_unpack(f2_mul(x2, f2_splat(2.0f * LOG2E * in)), e0, e1);
            f2_unpack(f2_add(f2_pack(ex2f(e0), ex2f(e1)), f2_splat(1.0f)), e0, e1);
            f2_unpack(f2_fma(f2_pack(rcpf(e0), rcpf(e1)), f2_splat(-2.0f * cap2), f2_splat(cap2)), e0, e1);
            x[t] = FORM == EACH && fabsf(y0) <= 1.0f ? x[t] : e0;
            x[t + 1] = FORM == EACH && fabsf(y1) <= 1.0f ? x[t + 1] : e1;
        }
    }
}
CEB_DEV float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
CEB_DEV uint32_t pack(float a, float b, __half) { return h2_as_u32(__floats2half2_rn(a, b)); }
CEB_DEV uint32_t pack(float a, float b, __nv_bfloat16) {
    __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&r);
}
// Whether a wait that began at clock t0 is over without its barrier: another role gave up, or
// the time is up (about a second, with no row computed again meanwhile), which is recorded with the
// barrier's number.
__device__ __noinline__ bool wait_over(volatile int* abort, int* err, uint32_t t0, int barrier) {
    if (*abort) return true;
    const uint32_t now = (uint32_t)clock(), limit = (uint32_t)CEB_WAIT_LIMIT_CYCLES;
    if (now - t0 < limit || now - (uint32_t)abort[1] < limit) return false;
    *abort = 1;
    if (err) atomicCAS(err, 0, (int)CEB_DEVERR_TIMEOUT_MMA | ((barrier + 1) << 16));
    return true;
}
// The pair's values, for sums that add the weights as rounded: a row's weights, as P V takes them,
// then still add up to one.  Adding them before the rounding leaves the output up to 1.4
// (fp16) or 1.5 (bf16) times as far off as its own rounding when the maximum in use is not the row's last
// one.  Here bf16 weights are added as rounded (3 % of the time, two bit operations a pair) and
// fp16 ones are not (converting them back took 9 %).
CEB_DEV f32x2 unpack(uint32_t u, __half) {
    const float2 f = __half22float2(u32_as_h2(u));
    return f2_pack(f.x, f.y);
}
CEB_DEV f32x2 unpack(uint32_t u, __nv_bfloat16) { return f2_pack(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
// MN-major operand, 128-byte swizzle: parts of 64 values along N `part` bytes apart, rows of
// 128 B along K in groups of eight.
CEB_DEV uint64_t v_desc(uint32_t saddr, uint32_t part) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
    d |= (uint64_t)(part >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
template <typename T>
CEB_DEV uint32_t mma_desc(int n) {
    return idesc_f16_f32(QT, n) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10));
}
// The bits of a 32-key piece that starts `at` keys into the row's frame: keys lo <= j < hi.
CEB_DEV uint32_t span_bits(int lo, int hi, int at) {
    const int a = min(max(lo - at, 0), 32), b = min(max(hi - at, 0), 32);
    const uint32_t up = b >= 32 ? 0xffffffffu : (1u << b) - 1u, dn = a >= 32 ? 0xffffffffu : (1u << a) - 1u;
    return up & ~dn;
}

// Products of 16 keys, the first of them d0 behind the row's place, into scores in log2 units.
CEB_DEV void score_piece(const Args& a, uint32_t (&v)[16], int d0, float scale2, float slope2, const float* table) {
    if (a.cap > 0.0f) {
        float* x = reinterpret_cast<float*>(v);
        if (a.cap <= SMALL_CAP) capped<FAR, 16>(x, a.scale / a.cap, scale2, a.cap * LOG2E);
        else capped<EACH, 16>(x, a.scale / a.cap, scale2, a.cap * LOG2E);
    } else {
#pragma unroll
        for (int t = 0; t < 16; ++t) v[t] = __float_as_uint(__uint_as_float(v[t]) * scale2);
    }
    if (a.slopes) {
        const float d = (float)d0;
#pragma unroll
        for (int t = 0; t < 16; ++t)
            v[t] = __float_as_uint(fmaf(slope2, fabsf(d + (float)t), __uint_as_float(v[t])));
    }
    if (table) {
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const float b = __ldg(table + min(max(d0 + t, -a.radius), a.radius)), b2 = b * LOG2E;
            // the lowest numbers stay numbers: -inf alone hides
            v[t] = __float_as_uint(__uint_as_float(v[t]) + (b2 == -INFINITY && b != -INFINITY ? -3.402823466e38f : b2));
        }
    }
}
// The same on a row's registers, N products from key distance d0 on, one form each.
// slopes: on one side of the diagonal the bias is linear in the key (side: keys before (-1) or
// behind (1) the place of every row of the warp, 0 mixed).
template <int N>
CEB_DEV void scores_slopes(uint32_t (&v)[N], int d0, int side, float scale2, float slope2) {
    if (side != 0) {
        const float c = side < 0 ? -slope2 : slope2;
        const f32x2 s2 = f2_splat(scale2), c2 = f2_splat(c), b2 = f2_splat(c * (float)d0);
#pragma unroll
        for (int t = 0; t < N; t += 2) {
            float x, y;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(v[t]), __uint_as_float(v[t + 1])), s2,
                             f2_fma(f2_pack((float)t, (float)(t + 1)), c2, b2)), x, y);
            v[t] = __float_as_uint(x);
            v[t + 1] = __float_as_uint(y);
        }
    } else {
        // slope2 |j - i'| = |slope2 (j - i')| with slope2's sign
        const uint32_t sign = __float_as_uint(slope2) & 0x80000000u;
        const f32x2 s2 = f2_splat(scale2), c2 = f2_splat(slope2), b2 = f2_splat(slope2 * (float)d0);
#pragma unroll
        for (int t = 0; t < N; t += 2) {
            float x, y;
            f2_unpack(f2_fma(f2_pack((float)t, (float)(t + 1)), c2, b2), x, y);
            x = __uint_as_float((__float_as_uint(x) & 0x7fffffffu) | sign);
            y = __uint_as_float((__float_as_uint(y) & 0x7fffffffu) | sign);
            f2_unpack(f2_fma(f2_pack(__uint_as_float(v[t]), __uint_as_float(v[t + 1])), s2, f2_pack(x, y)), x, y);
            v[t] = __float_as_uint(x);
            v[t + 1] = __float_as_uint(y);
        }
    }
}
// A row's scores capped, where all of the warp's products are below the cap.  False (v as it was) if not:
// prepare_capped then has the same bits for those that are.  4 x 4096 rows, 12 heads of 64: 623 us, where
// scores pass the cap 896.  (FAR alone for these, by each row's own choice, would take 790, but its code
// made the usual case 4 to 9 % slower.)
template <int N>
CEB_DEV bool scores_capped(uint32_t (&v)[N], float in, float scale2, float cap2) {
    float* x = reinterpret_cast<float*>(v);
    float top = 0.0f;
#pragma unroll
    for (int t = 0; t < N; t += 2) top = max3(top, fabsf(x[t]), fabsf(x[t + 1]));
    if (!__all_sync(0xffffffffu, top * in <= 1.0f)) return false;
    capped<NEAR, N>(x, in, scale2, cap2);
    return true;
}
// Bias by distance from the head's table.  False (v then holds nothing) if an entry times log2 e
// passes the lowest number.
template <int N>
CEB_DEV bool scores_table(uint32_t (&v)[N], int d0, int radius, float scale2, const float* table) {
    float low = 0.0f;
    const bool far = d0 >= radius || d0 + N - 1 <= -radius, inner = d0 >= -radius && d0 + N - 1 <= radius;
    if (__all_sync(0xffffffffu, far)) {
        const float b = __ldg(table + (d0 > 0 ? radius : -radius)) * LOG2E;
        low = b;
        const f32x2 s2 = f2_splat(scale2), b2 = f2_splat(b);
#pragma unroll
        for (int t = 0; t < N; t += 2) {
            float x, y;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(v[t]), __uint_as_float(v[t + 1])), s2, b2), x, y);
            v[t] = __float_as_uint(x);
            v[t + 1] = __float_as_uint(y);
        }
    } else if (__all_sync(0xffffffffu, inner)) {
        const float* p = table + d0;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const float b = __ldg(p + t) * LOG2E;
            low = fminf(low, b);
            v[t] = __float_as_uint(fmaf(__uint_as_float(v[t]), scale2, b));
        }
    } else {
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const float b = __ldg(table + min(max(d0 + t, -radius), radius)) * LOG2E;
            low = fminf(low, b);
            v[t] = __float_as_uint(fmaf(__uint_as_float(v[t]), scale2, b));
        }
    }
    return !__any_sync(0xffffffffu, low == -INFINITY);
}
// The masks of a chunk's keys for one row: bit t of word c is key k0 + 32 c + t.  doc < 0: the row
// sees none.
struct Words {
    uint32_t w[3];
};
template <int KC>
__device__ __noinline__ Words seen_chunk(const Args& a, const Seq& s, int place, int k0, int doc, const int* docs) {
    int lo, hi;
    window(a, s, place, lo, hi);
    if (doc < 0) hi = lo;
    const int prefix = doc < 0 ? 0 : s.prefix;
    Words r;
#pragma unroll
    for (int c = 0; c < KC / 32; ++c) {
        const int at = k0 + 32 * c;
        r.w[c] = (span_bits(lo, hi, at) | span_bits(0, prefix, at)) & span_bits(0, s.m, at);
        if (docs) {
            uint32_t same = 0;
#pragma unroll 8
            for (int t = 0; t < 32; ++t) same |= (uint32_t)(docs[32 * c + t] == doc) << t;
            r.w[c] &= same;
        }
    }
    return r;
}
// Scores of a chunk, prepared in TMEM 16 at a time: any combination.
template <int KC>
__device__ __noinline__ void prepare_scores(const Args& a, uint32_t s_t, int d0, float scale2, float slope2, const float* table) {
#pragma unroll 1
    for (int c = 0; c < KC; c += 16) {
        uint32_t v[16];
        tmem_ld16(s_t + (uint32_t)c, v);
        tmem_ld_wait();
        score_piece(a, v, d0 + c, scale2, slope2, table);
        tmem_st16(s_t + (uint32_t)c, v);
    }
    tmem_st_wait();
}

// Scores capped in TMEM 16 at a time, each by its own form.
template <int KC>
__device__ __noinline__ void prepare_capped(uint32_t s_t, float in, float scale2, float cap2) {
#pragma unroll 1
    for (int c = 0; c < KC; c += 16) {
        uint32_t v[16];
        tmem_ld16(s_t + (uint32_t)c, v);
        tmem_ld_wait();
        capped<EACH, 16>(reinterpret_cast<float*>(v), in, scale2, cap2);
        tmem_st16(s_t + (uint32_t)c, v);
    }
    tmem_st_wait();
}

// Weights for joining partial softmaxes, a lane each (`on`; maximum in log2 units and sum): f, the
// lane's factor, and for all lanes the joint maximum and sum.  Returns the lanes that have seen
// a key (of the others the O may be anything).
CEB_DEV unsigned join_weights(bool on, float2 ml, float& f, float& top, float& sum) {
    const bool none = !on || (ml.y == 0.0f && ml.x == -INFINITY);
    top = none ? -INFINITY : ml.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    f = none ? 0.0f : top == -INFINITY ? 1.0f : ex2f(ml.x - top);
    sum = none ? 0.0f : f * ml.y;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return __ballot_sync(0xffffffffu, !none);
}
// One row of the blocks of a cluster, by a warp: ml and o (fp32, HD values) lie at these places
// in every block.  A lane gets four values of the head, and the sum.
template <int HD, bool CLUSTER>
CEB_DEV void join_row(const float2* ml, const void* o, int parts, float (&acc)[4], float& sum) {
    const int lane = threadIdx.x & 31;
    auto at = [&](const void* p, int c) { return CLUSTER ? mapa_shared(smem_u32(p), c) : smem_u32(p); };
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                 : "=f"(v.x), "=f"(v.y)
                 : "r"(at(ml, min(lane, parts - 1)))
                 : "memory");
    float f, top;
    const unsigned used = join_weights(lane < parts, v, f, top, sum);
    acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
    for (int c0 = 0; c0 < parts; c0 += 4) {
        float4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (4 * lane < HD)
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(x[k].x), "=f"(x[k].y), "=f"(x[k].z), "=f"(x[k].w)
                             : "r"(at(o, min(c0 + k, parts - 1)) + 16 * lane)
                             : "memory");
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float fc = __shfl_sync(0xffffffffu, f, c0 + k);
            if (4 * lane < HD && (used >> (c0 + k) & 1u))
                acc[0] += fc * x[k].x, acc[1] += fc * x[k].y, acc[2] += fc * x[k].z, acc[3] += fc * x[k].w;
        }
    }
}

// SPLIT: the keys of an item are divided among the blocks of a cluster, which join their
// sums through distributed shared memory; one item a block.
// KIND: what stands between products and scores.  One of them is done in the registers that
// hold a row's products (PLAIN: the scale, in the exponentials' multiply-add); combinations, and
// scales that are not positive (the products' order is then not the scores'), take ANY, which
// prepares the scores in TMEM first.
enum { PLAIN, SLOPES, CAPPED, TABLE, ANY };

template <typename T, int HD, int KC_, int KIND, bool SPLIT>
__global__ void __launch_bounds__(NTHR, 2)
    attn_tile_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args a, int n_tiles, int n_kv, int n_items,
                     int batch, int parts) {
    using C = Cfg<HD, KC_>;
    constexpr int KC = C::KC, PC = KC / 32, NS = C::NS, ND = C::ND;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = base;
    uint8_t* sK = base + C::QB * C::Q_BYTES;
    uint8_t* sV = sK + NS * C::K_BYTES;
    Small& sm = *reinterpret_cast<Small*>(sV + NS * C::K_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_rows = QT / a.group;  // query rows of a tile
    const int part = SPLIT ? (int)cluster_ctarank() : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NBAR; ++i)
            mbar_init(smem_u32(&sm.bars[i]), (i == C::B_PFULL || i == C::B_PFULL + 1) ? 4 : (i == C::B_SFULL || i == C::B_SFULL + 1) ? 2 : (i >= C::B_IFREE ? 5 : 1));
        fence_mbar_init();
        sm.abort[0] = 0;
        sm.abort[1] = (int)clock();
        sm.now[0] = sm.now[1] = Chunk{0, 0, 0, 0};
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&qmap);
        tma_prefetch_desc(&kmap);
        tma_prefetch_desc(&vmap);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&sm.tmem), C::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    volatile int* abort = sm.abort;
    auto bar = [&](int i) { return smem_u32(&sm.bars[i]); };
    // Bounded waits; the error word names the barrier.  Most barriers are through when they are asked.
    auto wait_at = [&](int i, uint32_t par) {
        uint32_t t0 = 0;
        for (uint32_t n = 0; !mbar_try_wait(bar(i), par); ++n) {
            if (n == 0) t0 = (uint32_t)clock();
            if ((n & 255) == 255 && wait_over(abort, a.err, t0, i)) return false;
        }
        return true;
    };
    auto wait_warp = [&](int i, uint32_t par) { return __all_sync(0xffffffffu, wait_at(i, par)) != 0; };

    // A softmax thread holds a row of S: the control warps leave it registers.
    if (warp < 4) {
        regs_down<CONTROL_REGS>();
    }
    if (warp == 0) {
        // ------------------------------------------------ items, Q, and K / V of each chunk
        int g = 0, n_it = 0, n_ask = 0, n_q = 0;  // chunks, items, questions, items with keys
        int seq_k0 = -1, seq_m = -1;              // the sequence whose document ranges are kept
        bool ok = true;
        auto publish = [&](const Item& it) {
            const int r = n_it % NRING;
            if (n_it >= NRING && !wait_warp(C::B_IFREE + r, ((n_it / NRING) - 1) & 1)) return false;
            if (lane == 0) {
                sm.ring[r] = it;
                mbar_arrive(bar(C::B_IFULL + r));
            }
            __syncwarp();
            ++n_it;
            return true;
        };
        auto ask = [&] {
            if (lane == 0) {
                fence_proxy_async_smem();  // the last answer has been read
                mbar_arrive_expect_tx(bar(C::B_NEXT), 16);
                next_block_request(smem_u32(sm.answer), bar(C::B_NEXT));
            }
            __syncwarp();
            ++n_ask;
        };
        // A block stands for `batch` items side by side: lane l decodes item l, all lanes keep the
        // set of those that are queries of a sequence (tiles past a sequence's end cost nothing more).
        Item mine;
        unsigned todo;
        auto decode = [&](int block) {
            const int item = block * batch + lane;
            bool live = lane < batch && item < n_items;
            if (live) {
                const int tile = item % n_tiles, rest = item / n_tiles, seq = rest / n_kv;
                mine.kvh = rest - seq * n_kv;
                mine.i0 = tile * tile_rows;
                mine.empty = 1;
                live = load_seq(a, seq, tile == 0 && mine.kvh == 0, mine.s) && mine.i0 < mine.s.n;
            }
            todo = __ballot_sync(0xffffffffu, live);
        };
        int block = SPLIT ? (int)(blockIdx.x / parts) : (int)blockIdx.x;
        decode(block);
        if constexpr (!SPLIT) ask();
        while (ok) {
            if (!todo) {
                if (SPLIT) break;
                if (!(ok = wait_warp(C::B_NEXT, (n_ask - 1) & 1))) break;
                block = next_block_answer(smem_u32(sm.answer));
                __syncwarp();
                if (block < 0) break;
                ask();
                decode(block);
                continue;
            }
            const int from = __ffs(todo) - 1;
            todo &= todo - 1;
            Item it;
            it.kvh = __shfl_sync(0xffffffffu, mine.kvh, from);
            it.i0 = __shfl_sync(0xffffffffu, mine.i0, from);
            it.s.q0 = __shfl_sync(0xffffffffu, mine.s.q0, from);
            it.s.n = __shfl_sync(0xffffffffu, mine.s.n, from);
            it.s.k0 = __shfl_sync(0xffffffffu, mine.s.k0, from);
            it.s.m = __shfl_sync(0xffffffffu, mine.s.m, from);
            it.s.prefix = __shfl_sync(0xffffffffu, mine.s.prefix, from);
            const Seq& s = it.s;
            const int last = min(it.i0 + tile_rows, s.n) - 1, shift = s.m - s.n;
            int lo0, hi0, lo1, hi1;  // windows of the first and the last row: both ends rise with the row
            window(a, s, it.i0 + shift, lo0, hi0);
            window(a, s, last + shift, lo1, hi1);
            const int n1 = (s.prefix + KC - 1) / KC;  // chunks of the prefix, then those of the windows
            const int c0 = max(n1, lo0 / KC);
            const int total = n1 + (hi1 > lo0 ? max((hi1 + KC - 1) / KC - c0, 0) : 0);
            const int t_end = SPLIT ? (int)((int64_t)total * (part + 1) / parts) : total;
            int t = SPLIT ? (int)((int64_t)total * part / parts) : 0;
            // A bias by distance is greatest near the row's place as a rule: its chunk comes first, so that
            // the maxima are found at once and O is not rescaled chunk by chunk on the way there (texts
            // of 32 to 512 keys, slopes up to 0.1: 357 -> 349 us; 4 x 4096: 447 -> 400 us).
            int turn = 0;
            if (!SPLIT && (a.slopes || a.table) && total > 0) {
                const int near = max((it.i0 + last) / 2 + shift, 0) / KC;
                turn = min(near < c0 ? near : n1 + near - c0, total - 1);
                if (near < c0 && near >= n1) turn = 0;
            }
            auto chunk_at = [&](int p) {  // position -> chunk
                p += turn;
                p -= p >= total ? total : 0;
                return p < n1 ? p : c0 + p - n1;
            };
            int dq0 = INT32_MAX, dq1 = -1;  // documents of the tile's rows
            bool q_none = false;            // a row is of none
            if (a.doc_q) {
                for (int i = it.i0 + lane; i <= last; i += 32) {
                    const int d = a.doc_q[s.q0 + i];
                    if (d >= 0) dq0 = min(dq0, d), dq1 = max(dq1, d);
                    else q_none = true;
                }
                q_none = __any_sync(0xffffffffu, q_none) != 0;
                dq0 = __reduce_min_sync(0xffffffffu, dq0);
                dq1 = __reduce_max_sync(0xffffffffu, dq1);
            }
            // The next of the positions from `at` on whose chunk holds a document of the tile.  Ranges of
            // eight chunks are found at a time and kept for the sequence's other tiles and heads.  A slot
            // serves every 256th chunk and may change hands as the search goes on, so a lane takes its
            // position's range into registers while the slot is known to hold it.
            unsigned hits = 0;  // those of positions from hits_at on
            int hits_at = -32;
            int2 docs_of = make_int2(0, 0);  // of the chunk at position hits_at + lane
            auto seek = [&](int at) {
                if (at < hits_at + 32) {
                    const unsigned ahead = hits >> (at - hits_at);
                    if (ahead) return at + __ffs(ahead) - 1;
                    at = hits_at + 32;
                }
                if (s.k0 != seq_k0 || s.m != seq_m) {
                    seq_k0 = s.k0, seq_m = s.m;
                    if (lane < RANGES / 8) sm.range_tag[lane] = -1;
                    __syncwarp();
                }
                for (; at < t_end; at += 32) {
                    const int p = at + lane, c = chunk_at(p < t_end ? p : at);  // this lane's chunk
                    // A lane takes its range as soon as its slot holds it, then blocks of eight that are not
                    // there are fetched: the first waiting lane's each time, so 32 at most.  (Where positions
                    // jump from the prefix to the windows or wrap at the end, two lanes may want one slot for
                    // blocks of their own; both there at once they never are.)
                    bool want = p < t_end;
                    for (const int tag = c >> 3;;) {
                        if (want && sm.range_tag[tag % (RANGES / 8)] == tag) {
                            docs_of = sm.range[c % RANGES];
                            want = false;
                        }
                        const unsigned need = __ballot_sync(0xffffffffu, want);
                        if (!need) break;
                        __syncwarp();  // the slots have been read
                        const int b = __shfl_sync(0xffffffffu, tag, __ffs(need) - 1);
                        int d[8][KC / 32];
#pragma unroll
                        for (int x = 0; x < 8; ++x)
#pragma unroll
                            for (int y = 0; y < KC / 32; ++y) {
                                const int j = (8 * b + x) * KC + 32 * y + lane;
                                d[x][y] = j < s.m ? a.doc_k[s.k0 + j] : -1;
                            }
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            int mn = INT32_MAX, mx = -1, none = 0;
#pragma unroll
                            for (int y = 0; y < KC / 32; ++y) {
                                none |= d[x][y] < 0;
                                mn = d[x][y] < 0 ? mn : min(mn, d[x][y]);
                                mx = max(mx, d[x][y]);
                            }
                            mn = __reduce_min_sync(0xffffffffu, mn);
                            mx = __reduce_max_sync(0xffffffffu, mx);
                            if (__any_sync(0xffffffffu, none)) mx = -1 - max(mx, 0);
                            if (lane == 0) sm.range[(8 * b + x) % RANGES] = make_int2(mn, mx);
                        }
                        if (lane == 0) sm.range_tag[b % (RANGES / 8)] = b;
                        __syncwarp();
                    }
                    hits = __ballot_sync(
                        0xffffffffu, p < t_end && docs_of.x <= dq1 && (docs_of.y < 0 ? -1 - docs_of.y : docs_of.y) >= dq0);
                    hits_at = at;
                    if (hits) return at + __ffs(hits) - 1;
                }
                return max(at, t_end);
            };
            // positions t .. t_end - 1; a chunk is loaded once it is known whether another follows
            const int qb = n_q % C::QB;
            int pend = -1;                   // the chunk to load
            int2 pend_docs = docs_of;        // and its range of documents
            for (bool more = true; more; ++t) {
                int2 t_docs = docs_of;
                if (a.doc_k) {
                    t = seek(t);
                    t_docs.x = __shfl_sync(0xffffffffu, docs_of.x, t - hits_at);  // (no chunk at t_end: not used)
                    t_docs.y = __shfl_sync(0xffffffffu, docs_of.y, t - hits_at);
                }
                more = t < t_end;
                const int k0 = more ? chunk_at(t) * KC : 0;
                if (pend < 0) {  // the first chunk, or that there is none
                    it.empty = !more;
                    if (!(ok = publish(it))) break;
                    if (!more) break;
                    if (n_q >= C::QB && !(ok = wait_warp(C::B_QFREE + qb, ((n_q / C::QB) - 1) & 1))) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar(C::B_QFULL + qb), tile_rows * a.group * 128 * (HD / 64));
#pragma unroll
                        for (int x = 0; x < HD / 64; ++x)
                            tma_load_3d(smem_u32(sQ + qb * C::Q_BYTES + x * QT * 128), &qmap, bar(C::B_QFULL + qb), 64 * x,
                                        it.kvh * a.group, s.q0 + it.i0);
                    }
                    __syncwarp();
                    ++n_q;
                } else {
                    const int st = g % NS, ds = g % ND, j0 = pend;
                    if (g >= NS && !(ok = wait_warp(C::B_KFREE + st, ((g / NS) - 1) & 1))) break;
                    // (the description's slot: its last chunk, g - NS - 2, was done with before S of chunk g - NS)
                    int flags = (more ? 0 : LAST) | (j0 + KC > s.m ? TAIL : 0), docs = 0;
                    if (j0 + KC > s.m || !(j0 + KC <= s.prefix || (j0 >= lo1 && j0 + KC <= hi0))) flags |= MASKED;
                    if (a.doc_k) {
                        if (pend_docs.x == pend_docs.y) {  // keys of one document
                            docs = pend_docs.x;
                            if (q_none || dq0 != dq1 || dq0 != docs) flags |= MASKED | ONE_DOC;
                        } else {
                            docs = ds;
                            flags |= MASKED | DOCS;
#pragma unroll
                            for (int x = 0; x < KC / 32; ++x) {
                                const int j = j0 + 32 * x + lane;
                                sm.docs[ds][32 * x + lane] = j < s.m ? a.doc_k[s.k0 + j] : -1;
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) {
                        sm.chunk[ds] = Chunk{j0, flags, min(KC / 16, (s.m - j0 + 15) / 16), docs};
                        mbar_arrive_expect_tx(bar(C::B_KFULL + st), C::K_BYTES);
#pragma unroll
                        for (int x = 0; x < HD / 64; ++x)
                            tma_load_3d(smem_u32(sK + st * C::K_BYTES + x * KC * 128), &kmap, bar(C::B_KFULL + st), 64 * x,
                                        it.kvh, s.k0 + j0);
                    }
                    __syncwarp();
                    ++g;
                    if (g > NS && !(ok = wait_warp(C::B_VFREE + st, (((g - 1) / NS) - 1) & 1))) break;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar(C::B_VFULL + st), C::K_BYTES);
#pragma unroll
                        for (int x = 0; x < HD / 64; ++x)
                            tma_load_3d(smem_u32(sV + st * C::K_BYTES + x * KC * 128), &vmap, bar(C::B_VFULL + st), 64 * x,
                                        it.kvh, s.k0 + j0);
                    }
                    __syncwarp();
                }
                pend = k0;
                pend_docs = t_docs;
            }
        }
        if (ok) {
            Item end = {};
            end.kvh = -1;
            publish(end);
        }
        // what is in flight lands before the block can exit
        if (lane == 0) {
            if (!ok && n_ask > 0) mbar_wait(bar(C::B_NEXT), (n_ask - 1) & 1, nullptr, nullptr, 0);
            for (int k = n_q > C::QB ? n_q - C::QB : 0; k < n_q; ++k)
                mbar_wait(bar(C::B_QFULL + k % C::QB), (k / C::QB) & 1, nullptr, nullptr, 0);
            for (int c = g > NS ? g - NS : 0; c < g; ++c) {
                mbar_wait(bar(C::B_KFULL + c % NS), (c / NS) & 1, nullptr, nullptr, 0);
                if (ok || c < g - 1) mbar_wait(bar(C::B_VFULL + c % NS), (c / NS) & 1, nullptr, nullptr, 0);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA: S and P V, each as soon as it can be
        // All lanes run along, one issues.
        const bool one = elect_one();
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const int n16 = (a.head_dim + 15) / 16;
        const uint32_t s_desc = mma_desc<T>(KC);
        const uint32_t o_desc = mma_desc<T>(16 * n16) | (1u << 16);  // B (V) MN-major
        int gs = 0, gp = 0, n_it = 0, n_q = 0;  // next S, next P V, items, items with keys
        bool end = false, have = false, need_q = false, first = false;
        uint32_t firsts = 0;      // bit g & 3: chunk g begins an item (its P V overwrites O)
        int steps_of[2] = {0, 0};  // 16-key steps of the chunks whose P V is to come
        auto test = [&](int i, uint32_t par) { return __all_sync(0xffffffffu, mbar_test(bar(i), par)) != 0; };
        auto issue_s = [&] {
            const int st = gs % NS, qb = n_q % C::QB;
            const Chunk ck = sm.chunk[gs % ND];
            const bool last = (__shfl_sync(0xffffffffu, ck.flags, 0) & LAST) != 0;
            tc_fence_after();
            const uint32_t qs = smem_u32(sQ) + qb * C::Q_BYTES, ks = smem_u32(sK) + st * C::K_BYTES;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)  // 16 values of the head: 32 B of a 64-wide part
                mma_f16_ss_if(one && kk < n16, tm + (uint32_t)((gs & 1) * KC),
                              smem_desc_sw128(qs + (kk >> 2) * QT * 128) + (uint64_t)(2 * (kk & 3)),
                              smem_desc_sw128(ks + (kk >> 2) * KC * 128) + (uint64_t)(2 * (kk & 3)), s_desc, kk != 0);
            if (one) {
                mma_commit(bar(C::B_SFULL + (gs & 1)));
                mma_commit(bar(C::B_KFREE + st));
                if (last) mma_commit(bar(C::B_QFREE + qb));
                sm.now[gs & 1] = ck;
                mbar_arrive(bar(C::B_SFULL + (gs & 1)));
            }
            const int steps = __shfl_sync(0xffffffffu, ck.steps, 0);
            if (gs & 1) steps_of[1] = steps;
            else steps_of[0] = steps;
            firsts = (firsts & ~(1u << (gs & 3))) | (uint32_t)first << (gs & 3);
            first = false;
            ++gs;
            if (last) {
                have = false;
                ++n_q;
            }
        };
        auto issue_pv = [&] {
            const int st = gp % NS, steps = gp & 1 ? steps_of[1] : steps_of[0];
            tc_fence_after();
            const uint64_t vd = v_desc(smem_u32(sV) + st * C::K_BYTES, KC * 128);
            const bool over = firsts >> (gp & 3) & 1u;
#pragma unroll
            for (int j = 0; j < KC / 16; ++j)  // 16 keys: 2048 B of V, 8 columns of P
                mma_f16_ts_if(one && j < steps, tm + C::O_COL, tm + (uint32_t)((gp & 1) * KC + 8 * j),
                              vd + (uint64_t)(128 * j), o_desc, !(over && j == 0));
            if (one) {
                mma_commit(bar(C::B_PVDONE + (gp & 1)));
                mma_commit(bar(C::B_VFREE + st));
            }
            ++gp;
        };
        // S runs up to two chunks ahead of P V.  Of what a turn waits for, what comes first is asked first:
        // after P V of chunk g its end, which leaves S buffer g & 1 to chunk g + 2, then that chunk's K or
        // the weights of chunk g + 1, whichever is there.
        bool ok = true;
        uint32_t t0 = 0;
        for (uint32_t idle = 0; ok; ++idle) {
            if (gs - gp == 2 || (end && gp < gs)) {
                if (!(ok = wait_warp(C::B_PFULL + (gp & 1), (gp >> 1) & 1) && wait_warp(C::B_VFULL + gp % NS, (gp / NS) & 1))) break;
                issue_pv();
                if (!end && !(ok = wait_warp(C::B_PVDONE + ((gp - 1) & 1), ((gp - 1) >> 1) & 1))) break;
                idle = 0;
                continue;
            }
            if (end) break;
            if (!have && test(C::B_IFULL + n_it % NRING, (n_it / NRING) & 1)) {
                const volatile Item& it = sm.ring[n_it % NRING];
                const int kvh = __shfl_sync(0xffffffffu, it.kvh, 0), empty = __shfl_sync(0xffffffffu, it.empty, 0);
                __syncwarp();
                if (one) mbar_arrive(bar(C::B_IFREE + n_it % NRING));
                ++n_it;
                end = kvh < 0;
                have = need_q = first = !end && !empty;
                idle = 0;
                if (end) continue;
            }
            if (have && (!need_q || test(C::B_QFULL + n_q % C::QB, (n_q / C::QB) & 1)) &&
                test(C::B_KFULL + gs % NS, (gs / NS) & 1)) {
                need_q = false;
                issue_s();
                idle = 0;
                continue;
            }
            if (gp < gs && test(C::B_PFULL + (gp & 1), (gp >> 1) & 1) && test(C::B_VFULL + gp % NS, (gp / NS) & 1)) {
                issue_pv();
                if (!(ok = wait_warp(C::B_PVDONE + ((gp - 1) & 1), ((gp - 1) >> 1) & 1))) break;
                idle = 0;
                continue;
            }
            if (idle == 0) t0 = (uint32_t)clock();
            if ((idle & 255) == 255)  // bounded, as every wait
                ok = !__any_sync(0xffffffffu, wait_over(abort, a.err, t0, C::B_DRAIN));
        }
        if (one) mma_commit(bar(C::B_DRAIN));  // every MMA issued has finished before TMEM is freed
        mbar_wait(bar(C::B_DRAIN), 0, nullptr, nullptr, 0);
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------ softmax and output, thread = row
        regs_up<ROW_REGS>();
        const int qd = warp & 3;  // TMEM lanes 32 qd ..
        const int row = 32 * qd + lane;
        const uint32_t row_t = tmem + ((uint32_t)(32 * qd) << 16);
        const int qi = row / a.group, head_in = row - qi * a.group;
        const float scale2 = a.scale * LOG2E;
        // scores in log2 units are (products or prepared scores) * mul
        const float mul = KIND == PLAIN ? scale2 : 1.0f;
        int g = 0;
        bool ok = true;
        // V rows past the sequence's end hold other rows of the buffer: cleared
        auto clear_v = [&](int k0, int m) {
            const int st = g % NS;
            if (!wait_at(C::B_VFULL + st, (g / NS) & 1)) return false;
            if (row < KC && k0 + row >= m) {
#pragma unroll
                for (int x = 0; x < HD / 64; ++x)
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint4*>(sV + st * C::K_BYTES + (x * KC + row) * 128 + 16 * c) =
                            make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
            }
            return true;
        };
        for (int n_it = 0; ok; ++n_it) {
            const int r = n_it % NRING;
            if (!(ok = wait_warp(C::B_IFULL + r, (n_it / NRING) & 1))) break;
            // the item stays in the ring (released at its end): few of its numbers are worth a register
            const Item& it = sm.ring[r];
            if (it.kvh < 0) break;
            const Seq& s = it.s;
            const bool live = qi < tile_rows && it.i0 + qi < s.n;
            const int place = it.i0 + qi + s.m - s.n;
            const int doc = live && a.doc_q ? a.doc_q[s.q0 + it.i0 + qi] : 0;
            float slope2 = 0.0f;
            const float* table = nullptr;  // bias at distance 0
            if (KIND != PLAIN && live) {
                const int head = it.kvh * a.group + head_in;
                if (a.slopes) slope2 = -a.slopes[head] * LOG2E;
                if (a.table) table = a.table + (int64_t)head * (2 * (int64_t)a.radius + 1) + a.radius;
            }
            if (KIND >= TABLE && a.table && !table) table = a.table + a.radius;  // (a row that is none)
            const bool empty = it.empty;
            if (!__any_sync(0xffffffffu, live)) {
                // none of the warp's rows is one: it keeps to the barriers and its share of V
                for (bool last = empty; !last; ++g) {
                    if (!(ok = wait_warp(C::B_SFULL + (g & 1), (g >> 1) & 1))) break;
                    const Chunk ck = sm.now[g & 1];
                    last = (ck.flags & LAST) != 0;
                    if ((ck.flags & TAIL) && !(ok = clear_v(ck.k0, s.m))) break;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(C::B_PFULL + (g & 1)));
                    __syncwarp();
                }
                if (!ok) break;
                if constexpr (SPLIT) sm.ml[row] = make_float2(-INFINITY, 0.0f);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(C::B_IFREE + r));
                continue;
            }
            float m_run = -INFINITY, l_run = 0.0f;  // the maximum in use (log2 units) and the sum
            for (bool first = true; !empty; first = false) {
                // (a wait that failed shows at the chunk's end: what is computed then goes nowhere)
                ok = wait_at(C::B_SFULL + (g & 1), (g >> 1) & 1);
                tc_fence_after();
                const Chunk& ck = sm.now[g & 1];
                const int flags = ck.flags;
                const uint32_t s_t = row_t + (uint32_t)((g & 1) * KC);
                Words seen;
                if (flags & MASKED) {
                    if (flags & TAIL) ok &= clear_v(ck.k0, s.m);
                    seen = seen_chunk<KC>(a, s, place, ck.k0, (flags & ONE_DOC) && doc != ck.docs ? -1 : doc,
                                          flags & DOCS ? sm.docs[ck.docs] : nullptr);
                }
                const int d0 = KIND == PLAIN ? 0 : ck.k0 - place;
                if constexpr (KIND == ANY) prepare_scores<KC>(a, s_t, d0, scale2, slope2, table);
                uint32_t v[KC];
                auto load = [&] {
#pragma unroll
                    for (int pc = 0; pc < PC; ++pc)
                        tmem_ld32(s_t + (uint32_t)(32 * pc), reinterpret_cast<uint32_t(&)[32]>(v[32 * pc]));
                    tmem_ld_wait();
                };
                load();
                if constexpr (KIND == SLOPES) {
                    const int side = __all_sync(0xffffffffu, d0 >= 0) ? 1 : __all_sync(0xffffffffu, d0 + KC - 1 <= 0) ? -1 : 0;
                    scores_slopes(v, d0, side, scale2, slope2);
                }
                if constexpr (KIND == CAPPED)
                    if (!scores_capped(v, a.scale / a.cap, scale2, a.cap * LOG2E)) {
                        prepare_capped<KC>(s_t, a.scale / a.cap, scale2, a.cap * LOG2E);
                        load();
                    }
                if constexpr (KIND == TABLE)
                    if (!scores_table(v, d0, a.radius, scale2, table)) {
                        prepare_scores<KC>(a, s_t, d0, scale2, slope2, table);
                        load();
                    }
                if (flags & MASKED) {
#pragma unroll
                    for (int t = 0; t < KC; ++t)
                        if (!(seen.w[t / 32] >> (t % 32) & 1u)) v[t] = 0xff800000u;  // -inf
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int t = 0; t < KC; t += 2)
                    mx[(t >> 1) & 3] = max3(mx[(t >> 1) & 3], __uint_as_float(v[t]), __uint_as_float(v[t + 1]));
                float cm = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
                if (KIND == PLAIN) cm = cm == -INFINITY ? cm : cm * mul;  // (mul > 0)
                // A row raises its maximum for itself alone: other rows, be they of another sequence or none,
                // and keys that only they see have no part in its bits.
                const bool up = cm > m_run + RAISE<T>, raise = __any_sync(0xffffffffu, up && live);
                float alpha = 1.0f;
                if (up) {
                    alpha = ex2f(m_run - cm);
                    m_run = cm;
                }
                const f32x2 nm2 = f2_splat(UP<T> - (m_run == -INFINITY ? 0.0f : m_run)), mul2 = f2_splat(mul);
                f32x2 sum[2] = {f2_splat(0.0f), f2_splat(0.0f)};
#pragma unroll
                for (int pc = 0; pc < PC; ++pc) {
                    uint32_t pk[16];
#pragma unroll
                    for (int t = 0; t < 32; t += 2) {
                        float e0, e1;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(v[32 * pc + t]), __uint_as_float(v[32 * pc + t + 1])), mul2, nm2),
                                  e0, e1);
                        e0 = ex2f(e0);
                        e1 = ex2f(e1);
                        pk[t >> 1] = pack(e0, e1, T());
                        sum[(t >> 1) & 1] = f2_add(sum[(t >> 1) & 1],
                                                   std::is_same<T, __half>::value ? f2_pack(e0, e1) : unpack(pk[t >> 1], T()));
                    }
                    // the weights take the columns of scores that have been read
                    tmem_st16(s_t + (uint32_t)(16 * pc), pk);
                }
                {
                    float s0, s1;
                    f2_unpack(f2_add(sum[0], sum[1]), s0, s1);
                    l_run = l_run * alpha + (s0 + s1);
                }
                if (raise && !first) {  // O, once P V of chunk g - 1 has added to it
                    ok &= wait_at(C::B_PVDONE + ((g - 1) & 1), ((g - 1) >> 1) & 1);
                    tc_fence_after();
#pragma unroll 1
                    for (int o0 = 0; o0 < HD; o0 += 32) {
                        uint32_t ov[32];
                        tmem_ld32(row_t + C::O_COL + (uint32_t)o0, ov);
                        tmem_ld_wait();
#pragma unroll
                        for (int t = 0; t < 32; ++t) ov[t] = __float_as_uint(__uint_as_float(ov[t]) * alpha);
                        tmem_st32(row_t + C::O_COL + (uint32_t)o0, ov);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                if (!(ok = __all_sync(0xffffffffu, ok) != 0)) break;
                if (lane == 0) mbar_arrive(bar(C::B_PFULL + (g & 1)));
                ++g;
                if (flags & LAST) break;
            }
            // the item's last P V has finished: O / sum
            ok = ok && (empty || wait_warp(C::B_PVDONE + ((g - 1) & 1), ((g - 1) >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            if constexpr (SPLIT) {
                // this part's row, for the join: tiles of finished chunks make room for it
                float* o = reinterpret_cast<float*>(sK) + row * HD;
                sm.ml[row] = make_float2(m_run, l_run);
                if (!empty) {
#pragma unroll 1
                    for (int o0 = 0; o0 < HD; o0 += 32) {
                        uint32_t ov[32];
                        tmem_ld32(row_t + C::O_COL + (uint32_t)o0, ov);
                        tmem_ld_wait();
#pragma unroll
                        for (int t = 0; t < 32; t += 4)
                            *reinterpret_cast<uint4*>(o + o0 + t) = make_uint4(ov[t], ov[t + 1], ov[t + 2], ov[t + 3]);
                    }
                }
            } else {
                const float inv = l_run > 0.0f ? 1.0f / l_run : 0.0f;
                const int i = it.i0 + qi, head = it.kvh * a.group + head_in;
                T* out = static_cast<T*>(a.out) + (int64_t)(s.q0 + i) * a.o_row + head * a.o_head;
                f32x2 zero = f2_splat(0.0f);  // NaN once a value is no number or infinite
#pragma unroll 1
                for (int o0 = 0; o0 < a.head_dim; o0 += 32) {
                    uint32_t ov[32];
                    if (empty) {
#pragma unroll
                        for (int t = 0; t < 32; ++t) ov[t] = 0u;
                    } else {
                        tmem_ld32(row_t + C::O_COL + (uint32_t)o0, ov);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int t = 0; t < 32; t += 8)
                        if (o0 + t < a.head_dim) {
                            uint32_t w[4];
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const f32x2 y = f2_pack(__uint_as_float(ov[t + 2 * c]), __uint_as_float(ov[t + 2 * c + 1]));
                                float a0, a1;
                                zero = f2_fma(y, f2_splat(0.0f), zero);
                                f2_unpack(f2_mul(y, f2_splat(inv)), a0, a1);
                                w[c] = pack(a0, a1, T());
                            }
                            if (live) *reinterpret_cast<uint4*>(out + o0 + t) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                }
                float z0, z1;
                f2_unpack(zero, z0, z1);
                const bool wrong = z0 + z1 != 0.0f || !(l_run < INFINITY);
                // rows that met inf or NaN, be it their own or a hidden key's
                for (unsigned b = __ballot_sync(0xffffffffu, live && wrong); b; b &= b - 1) {
                    const int l = __ffs(b) - 1;
                    __syncwarp();
                    warp_row<T>(a, s, __shfl_sync(0xffffffffu, i, l), __shfl_sync(0xffffffffu, head, l), abort + 1);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(C::B_IFREE + r));
        }
        if constexpr (SPLIT) {
            // Each block joins every parts-th row, a warp a row, a lane four values of the head.
            __syncwarp();
            cluster_sync();
            const int item = blockIdx.x / parts, tile = item % n_tiles, rest = item / n_tiles;
            const int seq = rest / n_kv, kvh = rest - seq * n_kv, i0 = tile * tile_rows;
            Seq s;
            if (load_seq(a, seq, false, s) && i0 < s.n) {
                const int rows = min(tile_rows, s.n - i0) * a.group;
                for (int r = part + parts * (warp - 4); r < rows; r += parts * 4) {
                    float acc[4], sum;
                    join_row<HD, true>(sm.ml + r, sK + r * HD * 4, parts, acc, sum);
                    const int i = i0 + r / a.group, head = kvh * a.group + r % a.group;
                    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
                    bool wrong = sum != sum || sum == INFINITY;
                    if (4 * lane < a.head_dim) {
    #pragma unroll
                        for (int k = 0; k < 4; ++k) wrong |= !(fabsf(acc[k]) < INFINITY);
                        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(s.q0 + i) * a.o_row + head * a.o_head +
                                                  4 * lane) =
                            make_uint2(pack(acc[0] * inv, acc[1] * inv, T()), pack(acc[2] * inv, acc[3] * inv, T()));
                    }
                    if (__any_sync(0xffffffffu, wrong)) {
                        __syncwarp();
                        warp_row<T>(a, s, i, head);
                    }
                }
            }
        }
    }

    if constexpr (SPLIT) {
        __syncwarp();
        if (warp < 4) cluster_sync();
        cluster_sync();  // no block of the cluster still reads this one's shared memory
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM_COLS);
    }
}

template <typename T, int HD, int KC, int KIND>
int launch_tiles(const Args& a, cudaStream_t st) {
    using C = Cfg<HD, KC>;
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    const int n_kv = a.n_head / a.group, tile_rows = QT / a.group;
    const int n_tiles = (a.max_q + tile_rows - 1) / tile_rows;
    const int64_t items = (int64_t)n_tiles * n_kv * a.n_seqs;
    if (items > INT32_MAX / 8) return ceb_set_error(2, "attention_masked: %lld query tiles", (long long)items);
    CUtensorMap qmap, kmap, vmap;
    if (int rc = ceb_make_tmap_heads(&qmap, a.q, bf16, a.head_dim, a.n_head, a.q_rows, a.q_head, a.q_row, a.group, tile_rows))
        return rc;
    // (without key rows there is nothing to load: any map will do)
    const bool keys = a.k_rows > 0;
    if (int rc = ceb_make_tmap_heads(&kmap, keys ? a.k : a.q, bf16, a.head_dim, keys ? n_kv : a.n_head,
                                     keys ? a.k_rows : a.q_rows, keys ? a.k_head : a.q_head, keys ? a.k_row : a.q_row, 1,
                                     C::KC))
        return rc;
    if (int rc = ceb_make_tmap_heads(&vmap, keys ? a.v : a.q, bf16, a.head_dim, keys ? n_kv : a.n_head,
                                     keys ? a.k_rows : a.q_rows, keys ? a.v_head : a.q_head, keys ? a.v_row : a.q_row, 1,
                                     C::KC))
        return rc;
    // Few items with many keys: the keys of each are divided among a cluster, as long as that
    // fills the SMs and leaves each part some chunks.
    const int chunks = (a.max_k + C::KC - 1) / C::KC;
    int parts = 1;
    while (parts < 8 && items * parts * 2 <= 4 * ceb_num_sms() && chunks >= 4 * parts) parts *= 2;
    const size_t smem = smem_bytes<C>();
    cudaLaunchConfig_t cfg = {};
    // several items to a block where there are many: an item that is no query of its sequence
    // (ragged batches have a third of those) then costs a lane's look, not a block
    const int batch = parts > 1 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(32, items / (16 * ceb_num_sms())));
    cfg.gridDim = dim3((unsigned)((items + batch - 1) / batch * parts));
    cfg.blockDim = dim3(NTHR);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    auto kernel = parts > 1 ? attn_tile_kernel<T, HD, KC, KIND, true> : attn_tile_kernel<T, HD, KC, KIND, false>;
    if (int rc = ceb_func_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    cudaError_t e = cudaSuccess;
    CEB_LAUNCH(CEB_PROF_ATTN, st, 0.0, 0.0,
               e = cudaLaunchKernelEx(&cfg, kernel, qmap, kmap, vmap, a, n_tiles, n_kv, (int)items, batch, parts));
    CEB_CUDA_OK(e);
    return 0;
}

template <typename T, int HD>
int by_kind(const Args& a, cudaStream_t st) {
    if (!(a.scale > 0.0f) || (a.cap > 0.0f && (a.slopes || a.table))) return launch_tiles<T, HD, 64, ANY>(a, st);
    if (a.cap > 0.0f) return launch_tiles<T, HD, 64, CAPPED>(a, st);
    if (a.slopes) return launch_tiles<T, HD, 64, SLOPES>(a, st);
    if (a.table) return launch_tiles<T, HD, 64, TABLE>(a, st);
    // 96 keys a chunk where there are many and nothing but their products to turn into weights: 4 x 4096
    // rows, 12 heads of 64, 314 us (64 keys: 376 us).  Texts of 32 to 512 keys run out of them within a
    // chunk or two: 269 us with 64 (96: 304 us).
    if constexpr (HD == 64)
        if (a.max_k >= 1024) return launch_tiles<T, HD, 96, PLAIN>(a, st);
    return launch_tiles<T, HD, 64, PLAIN>(a, st);
}

}  // namespace
