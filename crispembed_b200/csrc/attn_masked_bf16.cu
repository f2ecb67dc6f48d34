// attn_masked_bf16.cu -- the masked attention kernels on bf16 values.
#include "attn_few.cuh"
#include "attn_tile.cuh"

int ceb_am::launch_bf16(const Args& a, cudaStream_t st) {
    if ((int64_t)a.max_q * a.group <= FROWS) return a.head_dim <= 64 ? launch_few<__nv_bfloat16, 64>(a, st) : launch_few<__nv_bfloat16, 128>(a, st);
    return a.head_dim <= 64 ? by_kind<__nv_bfloat16, 64>(a, st) : by_kind<__nv_bfloat16, 128>(a, st);
}
