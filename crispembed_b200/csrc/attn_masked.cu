// attn_masked.cu -- attention with shared key heads, score capping, a bias by distance and
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
constexpr int NS = 2;     // K / V stages
constexpr int NTHR = 256; // warp 0 loads, warp 1 TMEM + MMA, warps 4..7 softmax
constexpr int NRING = 4;  // items handed from the loading warp to the others

template <int HD>
struct Cfg {
    static constexpr int KC = HD == 64 ? 128 : 64;          // keys a chunk
    static constexpr int QB = HD == 64 ? 2 : 1;             // Q buffers
    static constexpr int Q_BYTES = QT * HD * 2;             // 64-wide parts, one behind the other
    static constexpr int K_BYTES = KC * HD * 2;
    static constexpr int STAGE = 2 * K_BYTES;               // K and V of a chunk
    static constexpr uint32_t S_COL = 0, P_COL = KC, O_COL = HD == 64 ? 192 : 128, TMEM_COLS = 256;
};
enum { B_QFULL, B_QFREE = B_QFULL + 2, B_FULL = B_QFREE + 2, B_EMPTY = B_FULL + NS, B_SFULL = B_EMPTY + NS, B_SFREE,
       B_PFULL, B_PVDONE, B_DRAIN, B_NEXT, B_IFULL, B_IEMPTY = B_IFULL + NRING, NBAR = B_IEMPTY + NRING };

// A decoded item: query rows i0 .. of the tile (local), its sequence, key head; `empty`: no
// key is seen by any row.  kvh < 0 ends the stream.
struct Item {
    Seq s;
    int i0, kvh, empty;
};
struct Chunk {
    int k0, flags;  // first key (local)
};
enum { LAST = 1, MASKED = 2, DOCS = 4 };

struct Small {  // shared memory behind the tiles
    uint64_t bars[NBAR];
    alignas(16) uint32_t answer[4];
    uint32_t tmem;
    int abort;
    Item ring[NRING];
    Chunk chunk[NS];
    int docs[NS][128];
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

template <int HD>
constexpr size_t smem_bytes() {
    return 1024 + Cfg<HD>::QB * Cfg<HD>::Q_BYTES + NS * Cfg<HD>::STAGE + sizeof(Small);
}
static_assert(2 * (smem_bytes<64>() + 1024) <= 228 * 1024 && 2 * (smem_bytes<128>() + 1024) <= 228 * 1024,
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
CEB_DEV uint32_t pack(float a, float b, __half) { return h2_as_u32(__floats2half2_rn(a, b)); }
CEB_DEV uint32_t pack(float a, float b, __nv_bfloat16) {
    __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&r);
}
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

// SPLIT: the keys of an item are divided among the blocks of a cluster, which join their
// sums through distributed shared memory; one item a block.
// GEN: scores are capped or biased (or their scale is not positive, so that the products'
// order is not the scores').
template <typename T, int HD, bool GEN, bool SPLIT>
__global__ void __launch_bounds__(NTHR, 2)
    attn_tile_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args a, int n_tiles, int n_kv, int n_items,
                     int parts) {
    using C = Cfg<HD>;
    constexpr int KC = C::KC, PC = KC / 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = base;
    uint8_t* sKV = base + C::QB * C::Q_BYTES;
    Small& sm = *reinterpret_cast<Small*>(sKV + NS * C::STAGE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_rows = QT / a.group;  // query rows of a tile
    const int part = SPLIT ? (int)cluster_ctarank() : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < NBAR; ++i)
            mbar_init(smem_u32(&sm.bars[i]), (i == B_SFREE || i == B_PFULL) ? 4 : (i >= B_IEMPTY ? 5 : 1));
        fence_mbar_init();
        sm.abort = 0;
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
    volatile int* abort = &sm.abort;
    auto bar = [&](int i) { return smem_u32(&sm.bars[i]); };
    auto wait_at = [&](int i, uint32_t par, int code) {
        return mbar_wait(bar(i), par, abort, a.err, code | ((i + 1) << 16));
    };
    auto wait_warp = [&](int i, uint32_t par, int code) { return __all_sync(0xffffffffu, wait_at(i, par, code)); };

    // A softmax thread holds a row of S: the control warps leave it registers.
    if (warp < 4) {
        regs_down<CONTROL_REGS>();
    }
    if (warp == 0) {
        // ------------------------------------------------ items, Q, and K / V of each chunk
        int g = 0, n_it = 0, n_ask = 0;
        bool ok = true;
        auto publish = [&](const Item& it) {
            const int r = n_it % NRING;
            if (n_it >= NRING && !wait_warp(B_IEMPTY + r, ((n_it / NRING) - 1) & 1, CEB_DEVERR_TIMEOUT_TMA))
                return false;
            if (lane == 0) {
                sm.ring[r] = it;
                mbar_arrive(bar(B_IFULL + r));
            }
            __syncwarp();
            ++n_it;
            return true;
        };
        auto ask = [&] {
            if (lane == 0) {
                fence_proxy_async_smem();  // the last answer has been read
                mbar_arrive_expect_tx(bar(B_NEXT), 16);
                next_block_request(smem_u32(sm.answer), bar(B_NEXT));
            }
            __syncwarp();
            ++n_ask;
        };
        int n_q = 0;  // items with keys: they take the Q buffers in turn
        int item = SPLIT ? (int)(blockIdx.x / parts) : (int)blockIdx.x;
        while (item >= 0 && item < n_items) {
            if constexpr (!SPLIT) ask();
            // item -> (sequence, key head, tile), tiles side by side
            Item it;
            const int tile = item % n_tiles, rest = item / n_tiles, seq = rest / n_kv;
            it.kvh = rest - seq * n_kv;
            it.i0 = tile * tile_rows;
            it.empty = 1;
            const bool live = load_seq(a, seq, tile == 0 && it.kvh == 0 && lane == 0, it.s) && it.i0 < it.s.n;
            if (live) {
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
                int dq0 = INT32_MAX, dq1 = -1;  // documents of the tile's rows
                if (a.doc_q) {
                    for (int i = it.i0 + lane; i <= last; i += 32) {
                        const int d = a.doc_q[s.q0 + i];
                        if (d >= 0) dq0 = min(dq0, d), dq1 = max(dq1, d);
                    }
                    dq0 = __reduce_min_sync(0xffffffffu, dq0);
                    dq1 = __reduce_max_sync(0xffffffffu, dq1);
                }
                // the next chunk from position `from` on that some row sees (t_end: none), its documents
                int kd[KC / 32], kd0 = 0, kd1 = 0;
                auto seek = [&](int from) {
                    if (!a.doc_k) return from;
                    for (; from < t_end; ++from) {
                        const int k0 = (from < n1 ? from : c0 + from - n1) * KC;
                        int mn = INT32_MAX, mx = -1, neg = 0;
#pragma unroll
                        for (int x = 0; x < KC / 32; ++x) {
                            const int j = k0 + 32 * x + lane;
                            kd[x] = j < s.m ? max(a.doc_k[s.k0 + j], -1) : -1;
                        }
#pragma unroll
                        for (int x = 0; x < KC / 32; ++x) {
                            if (kd[x] >= 0) mn = min(mn, kd[x]), mx = max(mx, kd[x]);
                            else if (k0 + 32 * x + lane < s.m) neg = 1;
                        }
                        kd0 = __reduce_min_sync(0xffffffffu, mn);
                        kd1 = __reduce_max_sync(0xffffffffu, mx);
                        if (__any_sync(0xffffffffu, neg)) kd0 = -1;  // (not one document)
                        if (kd1 >= 0 && kd1 >= dq0 && max(kd0, 0) <= dq1) break;
                    }
                    return from;
                };
                t = seek(t);
                it.empty = t >= t_end;
                if (!publish(it)) {
                    ok = false;
                    break;
                }
                if (!it.empty) {
                    const int qb = n_q % C::QB;
                    if (n_q >= C::QB && !wait_warp(B_QFREE + qb, ((n_q / C::QB) - 1) & 1, CEB_DEVERR_TIMEOUT_TMA)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar(B_QFULL + qb), tile_rows * a.group * 128 * (HD / 64));
#pragma unroll
                        for (int x = 0; x < HD / 64; ++x)
                            tma_load_3d(smem_u32(sQ + qb * C::Q_BYTES + x * QT * 128), &qmap, bar(B_QFULL + qb), 64 * x,
                                        it.kvh * a.group, s.q0 + it.i0);
                    }
                    __syncwarp();
                    ++n_q;
                    while (t < t_end) {
                        const int st = g % NS, k0 = (t < n1 ? t : c0 + t - n1) * KC;
                        if (g >= NS && !wait_warp(B_EMPTY + st, ((g / NS) - 1) & 1, CEB_DEVERR_TIMEOUT_TMA)) {
                            ok = false;
                            break;
                        }
                        const bool open = k0 + KC <= s.m && (k0 + KC <= s.prefix || (k0 >= lo1 && k0 + KC <= hi0));
                        int flags = open ? 0 : MASKED;
                        if (a.doc_k) {
                            flags |= MASKED | DOCS;
#pragma unroll
                            for (int x = 0; x < KC / 32; ++x) sm.docs[st][32 * x + lane] = kd[x];
                        }
                        const int next = seek(t + 1);
                        if (next >= t_end) flags |= LAST;
                        __syncwarp();
                        if (lane == 0) {
                            sm.chunk[st].k0 = k0;
                            sm.chunk[st].flags = flags;
                            mbar_arrive_expect_tx(bar(B_FULL + st), C::STAGE);
                            const uint32_t dst = smem_u32(sKV + st * C::STAGE);
#pragma unroll
                            for (int x = 0; x < HD / 64; ++x) {
                                tma_load_3d(dst + x * KC * 128, &kmap, bar(B_FULL + st), 64 * x, it.kvh, s.k0 + k0);
                                tma_load_3d(dst + C::K_BYTES + x * KC * 128, &vmap, bar(B_FULL + st), 64 * x, it.kvh,
                                            s.k0 + k0);
                            }
                        }
                        __syncwarp();
                        t = next;
                        ++g;
                    }
                    if (!ok) break;
                }
            }
            if constexpr (SPLIT) break;
            if (!(ok = wait_warp(B_NEXT, (n_ask - 1) & 1, CEB_DEVERR_TIMEOUT_TMA))) break;
            item = next_block_answer(smem_u32(sm.answer));
            __syncwarp();
        }
        if (ok) {
            Item end = {};
            end.kvh = -1;
            publish(end);
        }
        // what is in flight lands before the block can exit
        if (lane == 0) {
            if (!ok && n_ask > 0) mbar_wait(bar(B_NEXT), (n_ask - 1) & 1, nullptr, nullptr, 0);
            for (int k = n_q > C::QB ? n_q - C::QB : 0; k < n_q; ++k)
                mbar_wait(bar(B_QFULL + k % C::QB), (k / C::QB) & 1, nullptr, nullptr, 0);
            for (int c = g > NS ? g - NS : 0; c < g; ++c)
                mbar_wait(bar(B_FULL + c % NS), (c / NS) & 1, nullptr, nullptr, 0);
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA: S of chunk g, then P V of chunk g - 1
        if (lane == 0) {
            const int n16 = (a.head_dim + 15) / 16;
            const uint32_t s_desc = mma_desc<T>(KC);
            const uint32_t o_desc = mma_desc<T>(16 * n16) | (1u << 16);  // B (V) MN-major
            int g = 0, n_q = 0;
            bool ok = true, first_prev = false;
            auto issue_pv = [&](int gp, bool first) {
                const int sp = gp % NS;
                if (!wait_at(B_PFULL, gp & 1, CEB_DEVERR_TIMEOUT_MMA)) return false;
                tc_fence_after();
                const uint64_t vd = v_desc(smem_u32(sKV + sp * C::STAGE + C::K_BYTES), KC * 128);
#pragma unroll
                for (int j = 0; j < KC / 16; ++j)  // 16 keys: 2048 B of V, 8 columns of P
                    mma_f16_ts(tmem + C::O_COL, tmem + C::P_COL + (uint32_t)(8 * j), vd + (uint64_t)(128 * j), o_desc,
                               !(first && j == 0));
                mma_commit(bar(B_PVDONE));
                mma_commit(bar(B_EMPTY + sp));
                return true;
            };
            for (int n_it = 0; ok; ++n_it) {
                const int r = n_it % NRING;
                if (!(ok = wait_at(B_IFULL + r, (n_it / NRING) & 1, CEB_DEVERR_TIMEOUT_MMA))) break;
                const int kvh = *(volatile int*)&sm.ring[r].kvh, empty = *(volatile int*)&sm.ring[r].empty;
                mbar_arrive(bar(B_IEMPTY + r));
                if (kvh < 0) break;
                if (empty) continue;
                const int qb = n_q % C::QB;
                if (!(ok = wait_at(B_QFULL + qb, (n_q / C::QB) & 1, CEB_DEVERR_TIMEOUT_MMA))) break;
                ++n_q;
                const uint32_t qs = smem_u32(sQ + qb * C::Q_BYTES);
                for (bool first = true;; first = false) {
                    const int st = g % NS;
                    ok = wait_at(B_FULL + st, (g / NS) & 1, CEB_DEVERR_TIMEOUT_MMA) &&
                         (g == 0 || wait_at(B_SFREE, (g - 1) & 1, CEB_DEVERR_TIMEOUT_MMA));
                    if (!ok) break;
                    const bool last = (*(volatile int*)&sm.chunk[st].flags & LAST) != 0;
                    tc_fence_after();
                    const uint32_t ks = smem_u32(sKV + st * C::STAGE);
                    for (int kk = 0; kk < n16; ++kk)  // 16 values of the head: 32 B of a 64-wide part
                        mma_f16_ss(tmem + C::S_COL, smem_desc_sw128(qs + (kk >> 2) * QT * 128) + (uint64_t)(2 * (kk & 3)),
                                   smem_desc_sw128(ks + (kk >> 2) * KC * 128) + (uint64_t)(2 * (kk & 3)), s_desc, kk != 0);
                    mma_commit(bar(B_SFULL));
                    if (last) mma_commit(bar(B_QFREE + qb));
                    if (g > 0 && !(ok = issue_pv(g - 1, first_prev))) break;
                    first_prev = first;
                    ++g;
                    if (last) break;
                }
            }
            if (ok && g > 0) issue_pv(g - 1, first_prev);
            mma_commit(bar(B_DRAIN));  // every MMA issued has finished before TMEM is freed
            mbar_wait(bar(B_DRAIN), 0, nullptr, nullptr, 0);
        }
    } else if (warp >= 4) {
        // ------------------------------------------------ softmax and output, thread = row
        regs_up<ROW_REGS>();
        const int qd = warp & 3;  // TMEM lanes 32 qd ..
        const int row = 32 * qd + lane;
        const uint32_t row_t = tmem + ((uint32_t)(32 * qd) << 16);
        const int qi = row / a.group, head_in = row - qi * a.group;
        const float scale2 = a.scale * LOG2E;
        int g = 0;
        bool ok = true;
        // V rows past the sequence's end hold other rows of the buffer: cleared
        auto clear_v = [&](int st, int k0, int m) {
            if (k0 + KC > m && row < KC && k0 + row >= m) {
#pragma unroll
                for (int x = 0; x < HD / 64; ++x)
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint4*>(sKV + st * C::STAGE + C::K_BYTES + (x * KC + row) * 128 + 16 * c) =
                            make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
            }
        };
        for (int n_it = 0; ok; ++n_it) {
            const int r = n_it % NRING;
            if (!(ok = wait_warp(B_IFULL + r, (n_it / NRING) & 1, CEB_DEVERR_TIMEOUT_EPI))) break;
            // the item stays in the ring (released at its end): few of its numbers are worth a register
            const Item& it = sm.ring[r];
            if (it.kvh < 0) break;
            const Seq& s = it.s;
            const bool live = qi < tile_rows && it.i0 + qi < s.n;
            const int place = it.i0 + qi + s.m - s.n;
            const int doc = live && a.doc_q ? a.doc_q[s.q0 + it.i0 + qi] : 0;
            float slope2 = 0.0f;
            const float* table = nullptr;  // bias at distance 0
            if (GEN && live) {
                const int head = it.kvh * a.group + head_in;
                if (a.slopes) slope2 = -a.slopes[head] * LOG2E;
                if (a.table) table = a.table + (int64_t)head * (2 * (int64_t)a.radius + 1) + a.radius;
            }
            const bool empty = it.empty;
            if (!__any_sync(0xffffffffu, live)) {
                // none of the warp's rows is one: it keeps to the barriers and its share of V
                for (bool last = empty; !last; ++g) {
                    const int st = g % NS;
                    if (!(ok = wait_warp(B_SFULL, g & 1, CEB_DEVERR_TIMEOUT_EPI) &&
                               wait_warp(B_FULL + st, (g / NS) & 1, CEB_DEVERR_TIMEOUT_EPI)))
                        break;
                    last = (sm.chunk[st].flags & LAST) != 0;
                    clear_v(st, sm.chunk[st].k0, s.m);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(B_SFREE));
                    // (as the others: a phase of P V is waited for before the next may complete)
                    if (g > 0 && !(ok = wait_warp(B_PVDONE, (g - 1) & 1, CEB_DEVERR_TIMEOUT_EPI))) break;
                    if (lane == 0) mbar_arrive(bar(B_PFULL));
                    __syncwarp();
                }
                if (!ok) break;
                if constexpr (SPLIT) sm.ml[row] = make_float2(-INFINITY, 0.0f);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_IEMPTY + r));
                continue;
            }
            float m_run = -INFINITY, l_run = 0.0f;  // the maximum in use (log2 units) and the sum
            for (bool first = true; !empty; first = false) {
                const int st = g % NS;
                if (!(ok = wait_warp(B_SFULL, g & 1, CEB_DEVERR_TIMEOUT_EPI) &&
                           wait_warp(B_FULL + st, (g / NS) & 1, CEB_DEVERR_TIMEOUT_EPI)))
                    break;
                tc_fence_after();
                const int k0 = sm.chunk[st].k0, flags = sm.chunk[st].flags;
                uint32_t v[PC][32];
#pragma unroll
                for (int pc = 0; pc < PC; ++pc) tmem_ld32(row_t + C::S_COL + (uint32_t)(32 * pc), v[pc]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_SFREE));
                clear_v(st, k0, s.m);
                bool raise = false;
                float alpha = 1.0f;
                {
                    if constexpr (GEN) {
                        // scores in log2 units, each step a pass over the row's registers
                        if (a.cap > 0.0f) {
                            const float in = 2.0f * scale2 / a.cap, up = a.cap * LOG2E;
#pragma unroll
                            for (int pc = 0; pc < PC; ++pc)
#pragma unroll
                                for (int t = 0; t < 32; ++t) {
                                    // tanh y = 1 - 2 / (1 + e^2y)
                                    const float e = ex2f(__uint_as_float(v[pc][t]) * in);
                                    v[pc][t] = __float_as_uint(up * fmaf(-2.0f, rcpf(1.0f + e), 1.0f));
                                }
                        } else {
#pragma unroll
                            for (int pc = 0; pc < PC; ++pc)
#pragma unroll
                                for (int t = 0; t < 32; ++t)
                                    v[pc][t] = __float_as_uint(__uint_as_float(v[pc][t]) * scale2);
                        }
                        if (a.slopes) {
                            const float d0 = (float)(k0 - place);
#pragma unroll
                            for (int pc = 0; pc < PC; ++pc)
#pragma unroll
                                for (int t = 0; t < 32; ++t)
                                    v[pc][t] = __float_as_uint(
                                        fmaf(slope2, fabsf(d0 + (float)(32 * pc + t)), __uint_as_float(v[pc][t])));
                        }
                        if (table) {
                            const int d0 = k0 - place;
#pragma unroll
                            for (int pc = 0; pc < PC; ++pc)
#pragma unroll
                                for (int t = 0; t < 32; ++t) {
                                    const int d = min(max(d0 + 32 * pc + t, -a.radius), a.radius);
                                    const float b = __ldg(table + d), b2 = b * LOG2E;
                                    // the lowest numbers stay numbers: -inf alone hides
                                    v[pc][t] = __float_as_uint(__uint_as_float(v[pc][t]) +
                                                               (b2 == -INFINITY && b != -INFINITY ? -3.402823466e38f : b2));
                                }
                        }
                    }
                    if (flags & MASKED) {
#pragma unroll
                        for (int pc = 0; pc < PC; ++pc) {
                            int lo, hi;
                            window(a, s, place, lo, hi);
                            const int at = k0 + 32 * pc;
                            uint32_t w = (span_bits(lo, hi, at) | span_bits(0, s.prefix, at)) & span_bits(0, s.m, at);
                            if (flags & DOCS) {
                                uint32_t same = 0;
#pragma unroll
                                for (int t = 0; t < 32; ++t)
                                    same |= (uint32_t)(sm.docs[st][32 * pc + t] == doc) << t;
                                w &= doc >= 0 ? same : 0u;
                            }
#pragma unroll
                            for (int t = 0; t < 32; ++t)
                                if (!(w >> t & 1u)) v[pc][t] = 0xff800000u;  // -inf
                        }
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int pc = 0; pc < PC; ++pc)
#pragma unroll
                        for (int t = 0; t < 32; ++t) mx[t & 3] = fmaxf(mx[t & 3], __uint_as_float(v[pc][t]));
                    float cm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    if constexpr (!GEN) cm = cm == -INFINITY ? cm : cm * scale2;  // (scale > 0 here)
                    raise = __any_sync(0xffffffffu, cm > m_run + RAISE<T>) || first;
                    if (raise) {
                        const float m_new = fmaxf(m_run, cm);
                        alpha = m_new == -INFINITY ? 1.0f : ex2f(m_run - m_new);
                        m_run = m_new;
                    }
                    const float nm = UP<T> - (m_run == -INFINITY ? 0.0f : m_run);
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int pc = 0; pc < PC; ++pc)
#pragma unroll
                        for (int t = 0; t < 32; t += 2) {
                            const float x0 = __uint_as_float(v[pc][t]), x1 = __uint_as_float(v[pc][t + 1]);
                            float e0, e1;
                            if constexpr (GEN) {
                                e0 = ex2f(x0 + nm);
                                e1 = ex2f(x1 + nm);
                            } else {
                                e0 = ex2f(fmaf(x0, scale2, nm));
                                e1 = ex2f(fmaf(x1, scale2, nm));
                            }
                            sum[t & 2] += e0;
                            sum[(t & 2) + 1] += e1;
                            v[pc][t >> 1] = pack(e0, e1, T());  // (the pair's own registers or earlier ones)
                        }
                    l_run = l_run * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                }
                if (g > 0) {
                    // P V of chunk g - 1 has read P and added to O
                    if (!(ok = wait_warp(B_PVDONE, (g - 1) & 1, CEB_DEVERR_TIMEOUT_EPI))) break;
                    tc_fence_after();
                    if (raise && !first) {
#pragma unroll
                        for (int o0 = 0; o0 < HD; o0 += 32) {
                            uint32_t ov[32];
                            tmem_ld32(row_t + C::O_COL + (uint32_t)o0, ov);
                            tmem_ld_wait();
#pragma unroll
                            for (int t = 0; t < 32; ++t) ov[t] = __float_as_uint(__uint_as_float(ov[t]) * alpha);
                            tmem_st32(row_t + C::O_COL + (uint32_t)o0, ov);
                        }
                    }
                }
                {
#pragma unroll
                    for (int pc = 0; pc < PC; ++pc)
                        tmem_st16(row_t + C::P_COL + (uint32_t)(16 * pc), reinterpret_cast<const uint32_t(&)[16]>(v[pc]));
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(B_PFULL));
                ++g;
                if (flags & LAST) break;
            }
            // the item's last P V has finished: O / sum
            ok = ok && (empty || wait_warp(B_PVDONE, (g - 1) & 1, CEB_DEVERR_TIMEOUT_EPI));
            if (!ok) break;
            tc_fence_after();
            if constexpr (SPLIT) {
                // this part's row, for the join: tiles of finished chunks make room for it
                float* o = reinterpret_cast<float*>(sKV) + row * HD;
                sm.ml[row] = make_float2(m_run, l_run);
                if (!empty) {
#pragma unroll
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
                bool wrong = l_run != l_run || l_run == INFINITY;
                const int i = it.i0 + qi, head = it.kvh * a.group + head_in;
                T* out = static_cast<T*>(a.out) + (int64_t)(s.q0 + i) * a.o_row + head * a.o_head;
#pragma unroll
                for (int o0 = 0; o0 < HD; o0 += 32) {
                    uint32_t ov[32];
                    if (!empty) {
                        tmem_ld32(row_t + C::O_COL + (uint32_t)o0, ov);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int t = 0; t < 32; t += 8) {
                        if (o0 + t < a.head_dim) {
                            uint32_t w[4];
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                float x = __uint_as_float(ov[t + 2 * c]), y = __uint_as_float(ov[t + 2 * c + 1]);
                                if (empty) x = y = 0.0f;
                                wrong |= !(fabsf(x) < INFINITY) || !(fabsf(y) < INFINITY);
                                w[c] = pack(x * inv, y * inv, T());
                            }
                            if (live) *reinterpret_cast<uint4*>(out + o0 + t) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
                // rows that met inf or NaN, be it their own or a hidden key's
                for (unsigned b = __ballot_sync(0xffffffffu, live && wrong); b; b &= b - 1) {
                    const int l = __ffs(b) - 1;
                    __syncwarp();
                    warp_row<T>(a, s, __shfl_sync(0xffffffffu, i, l), __shfl_sync(0xffffffffu, head, l));
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(B_IEMPTY + r));
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
                const uint32_t ml = smem_u32(sm.ml), o = smem_u32(sKV);
                for (int r = part + parts * (warp - 4); r < rows; r += parts * 4) {
                    float top = -INFINITY;
                    for (int c = 0; c < parts; ++c) {
                        float m;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(m) : "r"(mapa_shared(ml + 8 * r, c)) : "memory");
                        top = fmaxf(top, m);
                    }
                    float sum = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int c = 0; c < parts; ++c) {
                        float m, l;
                        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                                     : "=f"(m), "=f"(l)
                                     : "r"(mapa_shared(ml + 8 * r, c))
                                     : "memory");
                        // a part without keys has no sums (its tiles hold anything)
                        if (l == 0.0f && m == -INFINITY) continue;
                        const float w = top == -INFINITY ? 1.0f : ex2f(m - top);
                        sum += w * l;
                        if (4 * lane < HD) {
                            float x[4];
                            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                                         : "r"(mapa_shared(o + (r * HD + 4 * lane) * 4, c))
                                         : "memory");
    #pragma unroll
                            for (int k = 0; k < 4; ++k) acc[k] += w * x[k];
                        }
                    }
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

template <typename T, int HD, bool GEN>
int launch_tiles(const Args& a, cudaStream_t st) {
    using C = Cfg<HD>;
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
    const size_t smem = smem_bytes<HD>();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * parts));
    cfg.blockDim = dim3(NTHR);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    auto kernel = parts > 1 ? attn_tile_kernel<T, HD, GEN, true> : attn_tile_kernel<T, HD, GEN, false>;
    if (int rc = ceb_func_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    cudaError_t e = cudaSuccess;
    CEB_LAUNCH(CEB_PROF_ATTN, st, 0.0, 0.0,
               e = cudaLaunchKernelEx(&cfg, kernel, qmap, kmap, vmap, a, n_tiles, n_kv, (int)items, parts));
    CEB_CUDA_OK(e);
    return 0;
}

template <typename T>
int launch(const Args& a, cudaStream_t st) {
    const bool gen = a.cap > 0.0f || a.slopes || a.table || !(a.scale > 0.0f);
    if (a.head_dim <= 64) return gen ? launch_tiles<T, 64, true>(a, st) : launch_tiles<T, 64, false>(a, st);
    return gen ? launch_tiles<T, 128, true>(a, st) : launch_tiles<T, 128, false>(a, st);
}

}  // namespace

extern "C" int ceb_attention_masked(const ceb_attn_params* p, const void* d_q, const void* d_k, const void* d_v,
                                    void* d_out, void* stream) {
    if (!p) return ceb_set_error(1, "attention_masked: no parameters");
    if (p->dtype != CEB_ACT_F16 && p->dtype != CEB_ACT_BF16)
        return ceb_set_error(1, "attention_masked: dtype %d unsupported (fp16 or bf16)", p->dtype);
    if (p->n_head <= 0 || p->n_head_kv <= 0 || p->n_head % p->n_head_kv || p->n_head / p->n_head_kv > 128)
        return ceb_set_error(1, "attention_masked: %d query heads on %d key heads", p->n_head, p->n_head_kv);
    if (p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8)
        return ceb_set_error(2, "attention_masked: head_dim %d (a multiple of 8 up to 128)", p->head_dim);
    if (p->n_seqs < 0 || p->q_rows < 0 || p->k_rows < 0 || p->max_q < 0 || p->max_k < 0)
        return ceb_set_error(1, "attention_masked: negative count");
    if (!std::isfinite(p->scale)) return ceb_set_error(1, "attention_masked: scale is not finite");
    if (!(p->softcap >= 0.0f) || !std::isfinite(p->softcap))
        return ceb_set_error(1, "attention_masked: softcap must be a finite number of at least 0");
    if (p->window_left < -1 || p->window_right < -1)
        return ceb_set_error(1, "attention_masked: window sides are -1 (open) or a distance");
    if (!p->d_doc_q != !p->d_doc_k) return ceb_set_error(1, "attention_masked: documents of one side only");
    if (p->d_slopes && p->d_rel_bias) return ceb_set_error(1, "attention_masked: slopes and a bias table");
    if (p->d_rel_bias && (p->rel_bias_radius < 0 || p->rel_bias_radius > (1 << 24)))
        return ceb_set_error(1, "attention_masked: bias radius %d", p->rel_bias_radius);
    if (p->n_seqs == 0 || p->q_rows == 0 || p->max_q == 0) return 0;
    if (!p->d_cu_q || !p->d_cu_k) return ceb_set_error(1, "attention_masked: row offsets missing");
    if (!d_q || !d_out || (p->k_rows > 0 && (!d_k || !d_v))) return ceb_set_error(1, "attention_masked: null tensor");
    if ((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v) |
         reinterpret_cast<uintptr_t>(d_out)) & 15)
        return ceb_set_error(1, "attention_masked: q, k, v and out must be 16-byte aligned");
    ceb_am::Args a = {};
    // strides: rows and heads of a tensor lie apart, at multiples of 16 bytes
    const int64_t hd = p->head_dim;
    constexpr int64_t FAR = (int64_t)1 << 38;    // a tensor map's strides end at 2^40 bytes
    constexpr int64_t WHOLE = (int64_t)1 << 45;  // more elements than any memory holds
    auto strides = [&](int64_t row, int64_t head, int rows, int heads, int64_t& r, int64_t& h, int64_t& span) {
        r = rows > 1 ? row : hd * heads;
        h = heads > 1 ? head : hd;
        if (r % 8 || h % 8 || r < hd || h < hd || r > FAR || h > FAR || r > WHOLE / rows || h > WHOLE / heads)
            return false;
        const int64_t in_row = (heads - 1) * h + hd;
        // rows hold their heads, or heads their rows (a single row or head has no other to run into)
        if (rows > 1 && heads > 1 && r < in_row && r > (h - hd) / (rows - 1)) return false;
        span = 2 * ((rows - 1) * r + in_row);
        return true;
    };
    int64_t span_q = 0, span_k = 0, span_v = 0, span_o = 0;
    if (!strides(p->q_row_stride, p->q_head_stride, p->q_rows, p->n_head, a.q_row, a.q_head, span_q) ||
        !strides(p->out_row_stride, p->out_head_stride, p->q_rows, p->n_head, a.o_row, a.o_head, span_o) ||
        (p->k_rows > 0 &&
         (!strides(p->k_row_stride, p->k_head_stride, p->k_rows, p->n_head_kv, a.k_row, a.k_head, span_k) ||
          !strides(p->v_row_stride, p->v_head_stride, p->k_rows, p->n_head_kv, a.v_row, a.v_head, span_v))))
        return ceb_set_error(1, "attention_masked: strides must be multiples of 8 that keep rows and heads apart");
    auto overlaps = [&](const void* x, int64_t span) {
        const uint8_t *b = static_cast<const uint8_t*>(x), *o = static_cast<const uint8_t*>(d_out);
        return span > 0 && b < o + span_o && o < b + span;
    };
    if (overlaps(d_q, span_q) || overlaps(d_k, span_k) || overlaps(d_v, span_v))
        return ceb_set_error(1, "attention_masked: out overlaps an input");
    a.q = d_q;
    a.k = d_k;
    a.v = d_v;
    a.out = d_out;
    a.cu_q = p->d_cu_q;
    a.cu_k = p->d_cu_k;
    a.prefix = p->d_prefix;
    a.doc_q = p->d_doc_q;
    a.doc_k = p->d_doc_k;
    a.slopes = p->d_slopes;
    a.table = p->d_rel_bias;
    a.n_head = p->n_head;
    a.group = p->n_head / p->n_head_kv;
    a.head_dim = p->head_dim;
    a.n_seqs = p->n_seqs;
    a.q_rows = p->q_rows;
    a.k_rows = p->k_rows;
    a.max_q = std::min(p->max_q, p->q_rows);
    a.max_k = p->max_k;
    a.left = p->window_left;
    a.right = p->window_right;
    a.radius = p->rel_bias_radius;
    a.scale = p->scale;
    a.cap = p->softcap;
    a.err = ceb_op_error_word();
    if (!a.err) return ceb_set_error(3, "attention_masked: device error word");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return p->dtype == CEB_ACT_F16 ? launch<__half>(a, st) : launch<__nv_bfloat16>(a, st);
}
