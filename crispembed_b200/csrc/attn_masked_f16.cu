// attn_masked_f16.cu -- the masked attention kernels on fp16 values.
#include "attn_tile.cuh"

int ceb_am::launch_f16(const Args& a, cudaStream_t st) {
    return a.head_dim <= 64 ? by_kind<__half, 64>(a, st) : by_kind<__half, 128>(a, st);
}
