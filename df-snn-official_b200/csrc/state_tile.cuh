// state_tile.cuh -- asynchronous staging of [steps, channels] tiles of a strided sequence.
#pragma once
#include "bulk_pipe.cuh"
#include "state_space.cuh"

namespace dfsnn {

// `bytes` of the BYTES at src to shared memory, zeros behind them
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, int bytes) {
    static_assert(BYTES == 4 || BYTES == 8 || BYTES == 16, "sizes that cp.async has");
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// A tile of ROWS steps x COLS neighbouring elements, by the NT threads of a block: steps from
// `rows` and elements from `cols` on become zero and are not read.  WIDE: rows start on 16-byte
// boundaries and are copied 16 bytes at a time.  Otherwise `words` says that all of them start on
// 4-byte boundaries; rows that do not (odd offsets of 16-bit types) are loaded and stored.
template <typename IO, int ROWS, int COLS, int NT, bool WIDE>
__device__ __forceinline__ void fill_tile(IO* dst, const IO* src, long long stride, int rows, int cols, bool words) {
    constexpr int E = (int)sizeof(IO);
    constexpr int BYTES = !WIDE ? 4 : COLS * E >= 16 ? 16 : COLS * E;
    constexpr int PER = BYTES / E, CPR = COLS / PER;
    if (WIDE || words) {
#pragma unroll
        for (int i0 = 0; i0 < ROWS * CPR; i0 += NT) {
            const int i = i0 + threadIdx.x, t = i / CPR, c = i % CPR * PER;
            if (ROWS * CPR % NT == 0 || i < ROWS * CPR) {
                int n = t < rows ? (cols - c) * E : 0;
                n = n < 0 ? 0 : n > BYTES ? BYTES : n;
                copy_async<BYTES>(dst + t * COLS + c, n ? src + t * stride + c : src, n);
            }
        }
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * COLS; i += NT) {
            const int t = i / COLS, c = i % COLS;
            dst[i] = t < rows && c < cols ? src[t * stride + c] : from_f<IO>(0.0f);
        }
    }
}

}  // namespace dfsnn
