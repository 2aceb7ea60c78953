// Kernels over paged caches with a scale per block of positions and head: attention, append, reading back.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "sp_host.h"
#include "sp_blocks.h"

namespace paged {
namespace {

template <class T, int KV>
void items_of(int HD, const BlockArgs &a, int grid, hipStream_t st) {
    if (HD == 128) hipLaunchKernelGGL((k_paged_attn<T, KV, 128>), dim3(grid), dim3(256), attn_smem<KV>, st, a);
    else hipLaunchKernelGGL((k_paged_attn<T, KV, 64>), dim3(grid), dim3(256), attn_smem<KV>, st, a);
}
template <class T>
void typed_items(bool i8, int HD, const BlockArgs &a, int grid, hipStream_t st) {
    if (i8) items_of<T, KV_I8_BLOCKS>(HD, a, grid, st);
    else items_of<T, KV_E4M3_BLOCKS>(HD, a, grid, st);
}
template <class T, int VEC, bool I8>
void append_codes(const BlockAppendArgs &a, int grid, size_t lds, hipStream_t st) {
    if (a.find) hipLaunchKernelGGL((k_append_blocks<T, VEC, I8, true>), dim3(grid), dim3(ROT_THREADS), lds, st, a);
    else hipLaunchKernelGGL((k_append_blocks<T, VEC, I8, false>), dim3(grid), dim3(ROT_THREADS), lds, st, a);
}
template <class T, int VEC>
void append_of(const BlockAppendArgs &a, int grid, size_t lds, hipStream_t st) {
    if (a.kv_dt == SP_DT_I8) append_codes<T, VEC, true>(a, grid, lds, st);
    else append_codes<T, VEC, false>(a, grid, lds, st);
}
template <class T>
void read_of(bool wide, const ReadArgs &a, hipStream_t st) {
    const int grid = (a.rows + a.per_block - 1) / a.per_block;
    if (wide) hipLaunchKernelGGL((k_paged_read<T, 8>), dim3(grid), dim3(ROT_THREADS), 0, st, a);
    else hipLaunchKernelGGL((k_paged_read<T, 1>), dim3(grid), dim3(ROT_THREADS), 0, st, a);
}

}  // namespace

void launch_block_items(int dtype, int kv_dtype, int HD, const BlockArgs &a, int grid, hipStream_t st) {
    const bool i8 = kv_dtype == SP_DT_I8;
    if (dtype == SP_DT_F16) typed_items<f16>(i8, HD, a, grid, st);
    else typed_items<bf16>(i8, HD, a, grid, st);
    HIPCHK(hipGetLastError());
}

void launch_block_append(int dtype, bool wide, const BlockAppendArgs &a, int query_blocks, size_t lds, hipStream_t st) {
    const int grid = a.chunks * 2 * a.splits + query_blocks;
    if (dtype == SP_DT_F32) { if (wide) append_of<float, 8>(a, grid, lds, st); else append_of<float, 1>(a, grid, lds, st); }
    else if (dtype == SP_DT_F16) { if (wide) append_of<f16, 8>(a, grid, lds, st); else append_of<f16, 1>(a, grid, lds, st); }
    else { if (wide) append_of<bf16, 8>(a, grid, lds, st); else append_of<bf16, 1>(a, grid, lds, st); }
    HIPCHK(hipGetLastError());
}

void launch_read(int dtype, bool wide, const ReadArgs &a, hipStream_t st) {
    if (dtype == SP_DT_F32) read_of<float>(wide, a, st);
    else if (dtype == SP_DT_F16) read_of<f16>(wide, a, st);
    else read_of<bf16>(wide, a, st);
    HIPCHK(hipGetLastError());
}

}  // namespace paged
