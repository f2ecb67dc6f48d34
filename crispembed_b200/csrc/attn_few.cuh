// attn_few.cuh -- masked attention for few rows a key head (single tokens): at most 16 query
// rows times query heads.
//
// A 128-row tile would be empty but for those rows, and its chain of barriers sets the pace: 55 us
// for the last tokens of 32 texts against up to 4096 keys, 16 heads of 128 on 4.  Here: 38 us, 4.0
// TB/s.  Every warp streams its own keys, 16 at a step, through a ring of its own in shared
// memory (cp.async, no barrier between warps): m16n8k16 products with the rows as M, one
// online softmax a warp, weights straight from the product's registers.  A product's 16 head
// values may be any 16 as long as Q and K agree, so K is read in 16-byte pieces as it lies.  The
// warps' sums, and those of the blocks of a cluster among which a sequence's keys are divided,
// meet at the end through (distributed) shared memory.  Bound by the keys' bytes.
#pragma once

#include "attn_tile.cuh"

namespace {

constexpr int FW = 4;        // warps a block
constexpr int FSTAGES = 3;   // steps in flight a warp
constexpr int FROWS = 16, FKEYS = 16;

CEB_DEV void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CEB_DEV void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes, or zeros (nothing is read then)
CEB_DEV void cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
CEB_DEV void ldmatrix_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Shared memory of a block: the warps' rings, which the warps' sums then take, and (maximum, sum).
template <int HD>
struct FewSmem {
    static constexpr int STEP = 2 * FKEYS * HD * 2;  // K and V of a step
    static constexpr int RING = FSTAGES * STEP;
    static_assert(RING >= FROWS * HD * 4, "a warp's O fits its ring");
    static constexpr size_t BYTES = (size_t)FW * RING + FW * FROWS * sizeof(float2);
};

template <typename T, int HD, bool SPLIT>
__global__ void __launch_bounds__(32 * FW, 2)
    attn_few_kernel(const __grid_constant__ Args a, int n_kv, int parts) {
    using S_ = FewSmem<HD>;
    constexpr int CH = HD / 8;  // 16-byte pieces of a row
    extern __shared__ __align__(128) uint8_t smem_raw[];
    float2* ml = reinterpret_cast<float2*>(smem_raw + FW * S_::RING);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int part = SPLIT ? (int)cluster_ctarank() : 0;
    const int item = SPLIT ? (int)(blockIdx.x / parts) : (int)blockIdx.x, seq = item / n_kv, kvh = item - seq * n_kv;
    Seq s;
    const bool live = load_seq(a, seq, kvh == 0 && part == 0 && threadIdx.x == 0, s) && s.n > 0;
    const int rows = live ? s.n * a.group : 0;  // <= FROWS (the launch sees to it)
    const uint32_t ring = smem_u32(smem_raw) + warp * S_::RING;
    if (live) {
        const T* kp = static_cast<const T*>(a.k) + (int64_t)s.k0 * a.k_row + kvh * a.k_head;
        const T* vp = static_cast<const T*>(a.v) + (int64_t)s.k0 * a.v_row + kvh * a.v_head;
        // this lane's two rows of the product: g and g + 8
        int place[2], lo[2], hi[2], doc[2];
        float slope2[2];
        const float* table[2];
        bool on[2];
        uint32_t q[HD / 16][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h, i = r / a.group, head = kvh * a.group + r % a.group;
            on[h] = r < rows;
            place[h] = i + s.m - s.n;
            window(a, s, place[h], lo[h], hi[h]);
            doc[h] = on[h] && a.doc_q ? a.doc_q[s.q0 + i] : 0;
            slope2[h] = on[h] && a.slopes ? -a.slopes[head] * LOG2E : 0.0f;
            table[h] = on[h] && a.table ? a.table + (int64_t)head * (2 * (int64_t)a.radius + 1) + a.radius : nullptr;
            const T* qr = static_cast<const T*>(a.q) + (int64_t)(s.q0 + i) * a.q_row + head * a.q_head;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {  // 16-byte pieces t, t + 4, ..: two products each
                uint4 u = make_uint4(0, 0, 0, 0);
                if (on[h] && 8 * (t + 4 * c) < a.head_dim) u = *reinterpret_cast<const uint4*>(qr + 8 * (t + 4 * c));
                q[2 * c][h] = u.x;
                q[2 * c][2 + h] = u.y;
                q[2 * c + 1][h] = u.z;
                q[2 * c + 1][2 + h] = u.w;
            }
        }
        // the block's steps of 16 keys, by position: those of the prefix, then those of the windows
        int lo0, hi0, lo1, hi1;
        window(a, s, s.m - s.n, lo0, hi0);
        window(a, s, s.m - 1, lo1, hi1);
        const int n1 = (s.prefix + FKEYS - 1) / FKEYS, c0 = max(n1, lo0 / FKEYS);
        const int total = n1 + (hi1 > lo0 ? max((hi1 + FKEYS - 1) / FKEYS - c0, 0) : 0);
        const int first = SPLIT ? (int)((int64_t)total * part / parts) : 0;
        const int end = SPLIT ? (int)((int64_t)total * (part + 1) / parts) : total;
        auto key_at = [&](int p) { return (p < n1 ? p : c0 + p - n1) * FKEYS; };
        // A row's piece c lies at c ^ f(row): a K read takes four pieces of two rows, a V read one of eight.
        // A lane copies one piece of every RS-th row.
        constexpr int RS = 32 / CH;
        const int fr = lane / CH, fc = lane % CH;
        const bool fin = 8 * fc < a.head_dim;
        const T* kl = kp + (int64_t)fr * a.k_row + (fin ? 8 * fc : 0);
        const T* vl = vp + (int64_t)fr * a.v_row + (fin ? 8 * fc : 0);
        auto fetch = [&](int p, int st) {
            if (p < end) {
                const int j0 = key_at(p);
                const uint32_t sk = ring + st * S_::STEP + fr * HD * 2, sv = sk + FKEYS * HD * 2;
                const T *ks = kl + j0 * a.k_row, *vs = vl + j0 * a.v_row;
#pragma unroll
                for (int x = 0; x < FKEYS / RS; ++x) {
                    const int r = RS * x + fr;
                    const bool in = fin && j0 + r < s.m;
                    cp16(sk + x * RS * HD * 2 + 16 * (fc ^ ((r & 1) << 2)), in ? ks : kp, in);
                    cp16(sv + x * RS * HD * 2 + 16 * (fc ^ (r & 7)), in ? vs : vp, in);
                    ks += RS * a.k_row;
                    vs += RS * a.v_row;
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        const int halves = rows > 8 ? 2 : 1;  // rows 8 .. 15 are there at all
        float o[HD / 8][4];
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
        const float scale2 = a.scale * LOG2E;
#pragma unroll
        for (int st = 0; st < FSTAGES - 1; ++st) fetch(first + warp + FW * st, st);
        int st = 0;
        for (int p = first + warp; p < end; p += FW) {
            fetch(p + FW * (FSTAGES - 1), st == 0 ? FSTAGES - 1 : st - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(FSTAGES - 1) : "memory");
            __syncwarp();
            const int j0 = key_at(p);
            const uint32_t sk = ring + st * S_::STEP, sv = sk + FKEYS * HD * 2;
            float c[2][4] = {};  // keys 0..7 and 8..15: (row g, keys 2t, 2t + 1), (row g + 8, the same)
#pragma unroll
            for (int x = 0; x < HD / 32; ++x)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int r = 8 * n + g;
                    uint4 b;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                                 : "r"(sk + r * HD * 2 + 16 * ((t + 4 * x) ^ ((r & 1) << 2)))
                                 : "memory");
                    mma_16816(c[n], q[2 * x], b.x, b.y, T());
                    mma_16816(c[n], q[2 * x + 1], b.z, b.w, T());
                }
            // scores in log2 units; keys that the row does not see are -inf
            float w[2][4];  // [row][key 2t, 2t + 1, 2t + 8, 2t + 9]
            const bool open = !a.doc_k && j0 + FKEYS <= s.m &&
                              (j0 + FKEYS <= s.prefix || (j0 >= lo1 && j0 + FKEYS <= hi0));  // every row sees them all
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= halves) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[h][e] = -INFINITY;
                    continue;
                }
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[h][e] = c[e >> 1][2 * h + (e & 1)];
                    const float in = a.scale / a.cap;
                    const float top = fmaxf(max3(fabsf(w[h][0]), fabsf(w[h][1]), fabsf(w[h][2])), fabsf(w[h][3]));
                    if (__all_sync(0xffffffffu, top * fabsf(in) <= 1.0f)) capped<NEAR, 4>(w[h], in, scale2, a.cap * LOG2E);
                    else capped<EACH, 4>(w[h], in, scale2, a.cap * LOG2E);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[h][e] = c[e >> 1][2 * h + (e & 1)] * scale2;
                }
                const int d0 = j0 + 2 * t - place[h];
                if (a.slopes) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) w[h][e] = fmaf(slope2[h], fabsf((float)(d0 + 8 * (e >> 1) + (e & 1))), w[h][e]);
                }
                if (table[h]) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float b = __ldg(table[h] + min(max(d0 + 8 * (e >> 1) + (e & 1), -a.radius), a.radius));
                        const float b2 = b * LOG2E;
                        w[h][e] += b2 == -INFINITY && b != -INFINITY ? -3.402823466e38f : b2;
                    }
                }
                if (!open) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int jk = j0 + 2 * t + 8 * (e >> 1) + (e & 1);
                        bool seen = on[h] && jk < s.m && (jk < s.prefix || (jk >= lo[h] && jk < hi[h]));
                        if (a.doc_k && seen) seen = doc[h] >= 0 && a.doc_k[s.k0 + jk] == doc[h];
                        w[h][e] = seen ? w[h][e] : -INFINITY;
                    }
                }
            }
            uint32_t pa[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= halves) {
                    pa[h] = pa[2 + h] = 0u;
                    continue;
                }
                float cm = fmaxf(fmaxf(w[h][0], w[h][1]), fmaxf(w[h][2], w[h][3]));
                cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, 1));
                cm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, 2));
                const float m_new = cm > m_run[h] + RAISE<T> || m_run[h] == -INFINITY ? fmaxf(m_run[h], cm) : m_run[h];
                if (__any_sync(0xffffffffu, m_new != m_run[h])) {
                    const float f = m_new == -INFINITY ? 1.0f : ex2f(m_run[h] - m_new);
                    l_run[h] *= f;
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) o[n][2 * h] *= f, o[n][2 * h + 1] *= f;
                    m_run[h] = m_new;
                }
                const float nm = UP<T> - (m_run[h] == -INFINITY ? 0.0f : m_run[h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[h][e] = ex2f(w[h][e] + nm);
                pa[h] = pack(w[h][0], w[h][1], T());
                pa[2 + h] = pack(w[h][2], w[h][3], T());
                float s0, s1;
                f2_unpack(f2_add(unpack(pa[h], T()), unpack(pa[2 + h], T())), s0, s1);
                l_run[h] += s0 + s1;
            }
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {  // 16 head values: four 8x8 tiles (keys 0-7, 8-15) x two pieces
                const int r = lane & 15, cc = 2 * n + (lane >> 4);
                uint32_t b[4];
                ldmatrix_t(sv + r * HD * 2 + 16 * (cc ^ (r & 7)), b);
                mma_16816(o[2 * n], pa, b[0], b[1], T());
                mma_16816(o[2 * n + 1], pa, b[2], b[3], T());
            }
            __syncwarp();
            st = st + 1 == FSTAGES ? 0 : st + 1;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        // this warp's sums take its ring
        float* os = reinterpret_cast<float*>(smem_raw + warp * S_::RING);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
            if (t == 0) ml[warp * FROWS + g + 8 * h] = make_float2(m_run[h], l_run[h]);
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
                *reinterpret_cast<float2*>(os + (g + 8 * h) * HD + 8 * n + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        }
    }
    __syncthreads();
    // The warps' sums into the first warp's place: a warp a row, a lane four values of the head.
    for (int r = warp; r < rows; r += FW) {
        float f, top, sum;
        const unsigned used = join_weights(lane < FW, ml[min(lane, FW - 1) * FROWS + r], f, top, sum);
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < FW; ++c) {
            const float fc = __shfl_sync(0xffffffffu, f, c);
            if (4 * lane < HD && (used >> c & 1u)) {
                const float4 x = *reinterpret_cast<const float4*>(smem_raw + c * S_::RING + (r * HD + 4 * lane) * 4);
                acc[0] += fc * x.x, acc[1] += fc * x.y, acc[2] += fc * x.z, acc[3] += fc * x.w;
            }
        }
        if (4 * lane < HD)
            *reinterpret_cast<float4*>(smem_raw + (r * HD + 4 * lane) * 4) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        __syncwarp();
        if (lane == 0) ml[r] = make_float2(top, sum);
    }
    if (SPLIT) cluster_sync();
    else __syncthreads();
    // Every parts-th row is this block's to finish.
    for (int r = part + parts * warp; r < rows; r += parts * FW) {
        float acc[4], sum;
        join_row<HD, SPLIT>(ml + r, smem_raw + r * HD * 4, parts, acc, sum);
        const int i = r / a.group, head = kvh * a.group + r % a.group;
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        bool wrong = !(sum < INFINITY);
        if (4 * lane < a.head_dim) {
#pragma unroll
            for (int k = 0; k < 4; ++k) wrong |= !(fabsf(acc[k]) < INFINITY);
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (int64_t)(s.q0 + i) * a.o_row + head * a.o_head + 4 * lane) =
                make_uint2(pack(acc[0] * inv, acc[1] * inv, T()), pack(acc[2] * inv, acc[3] * inv, T()));
        }
        if (__any_sync(0xffffffffu, wrong)) {  // inf or NaN, be it a hidden key's
            __syncwarp();
            warp_row<T>(a, s, i, head);
        }
    }
    if (SPLIT) cluster_sync();  // no block of the cluster still reads this one's shared memory
}

template <typename T, int HD>
int launch_few(const Args& a, cudaStream_t st) {
    const int n_kv = a.n_head / a.group;
    const int64_t items = (int64_t)n_kv * a.n_seqs;
    if (items > INT32_MAX / 8) return ceb_set_error(2, "attention_masked: %lld key heads", (long long)items);
    const int steps = (a.max_k + FKEYS - 1) / FKEYS;
    // Two blocks run on an SM; up to two waves of them are made, as long as a warp keeps four steps
    // (32 texts: one wave 37.5 us, two 37.8, four 47.6, when the blocks' beginnings and ends show;
    // a single text wants all it can get).
    int parts = 1;
    while (parts < 8 && items * parts * 2 <= 4 * ceb_num_sms() && steps >= 4 * FW * parts) parts *= 2;
    const size_t smem = FewSmem<HD>::BYTES;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * parts));
    cfg.blockDim = dim3(32 * FW);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    auto kernel = parts > 1 ? attn_few_kernel<T, HD, true> : attn_few_kernel<T, HD, false>;
    if (int rc = ceb_func_smem(reinterpret_cast<const void*>(kernel), smem)) return rc;
    cudaError_t e = cudaSuccess;
    CEB_LAUNCH(CEB_PROF_ATTN, st, 0.0, 0.0, e = cudaLaunchKernelEx(&cfg, kernel, a, n_kv, parts));
    CEB_CUDA_OK(e);
    return 0;
}

}  // namespace
