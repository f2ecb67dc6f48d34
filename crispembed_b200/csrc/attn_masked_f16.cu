// attn_masked_f16.cu -- the masked attention kernels on fp16 values.
#include "attn_few.cuh"
#include "attn_tile.cuh"

int ceb_am::launch_f16(const Args& a, cudaStream_t st) {
    if ((int64_t)a.max_q * a.group <= FROWS) return a.head_dim <= 64 ? launch_few<__half, 64>(a, st) : launch_few<__half, 128>(a, st);
    return a.head_dim <= 64 ? by_kind<__half, 64>(a, st) : by_kind<__half, 128>(a, st);
}
