// attn_masked.cu -- the C entry of masked attention: checks, then the kernels of attn_tile.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/ceb_ops.h"
#include "attn_masked.h"
#include "ceb_internal.h"

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
    // (what the kernels form of them, 2 scale log2(e) / softcap among it, stays finite)
    if (!(std::fabs(p->scale) <= 1e15f)) return ceb_set_error(1, "attention_masked: scale beyond 1e15");
    if (p->softcap != 0.0f && !(p->softcap >= 1e-15f && p->softcap <= 1e30f))
        return ceb_set_error(1, "attention_masked: softcap must be 0 or 1e-15 to 1e30");
    if (p->window_left < -1 || p->window_right < -1)
        return ceb_set_error(1, "attention_masked: window sides are -1 (open) or a distance");
    // (an empty side has no numbers to give)
    if (!p->d_doc_q != !p->d_doc_k && p->q_rows > 0 && p->k_rows > 0)
        return ceb_set_error(1, "attention_masked: documents of one side only");
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
    a.doc_q = p->k_rows > 0 ? p->d_doc_q : nullptr;
    a.doc_k = p->k_rows > 0 ? p->d_doc_k : nullptr;
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
    return p->dtype == CEB_ACT_F16 ? ceb_am::launch_f16(a, st) : ceb_am::launch_bf16(a, st);
}
