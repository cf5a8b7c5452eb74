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
// until all but the newest LEFT groups of this thread have landed
template <int LEFT>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// A tile of ROWS steps x COLS neighbouring elements, by the NT threads of a block: steps from `rows`
// and elements from `cols` on become zero and are not read.  WIDE: rows start on 16-byte
// boundaries and are copied 16 bytes at a time (8 where a row of the tile has no more).  Otherwise
// `words` says that every row starts on a 4-byte boundary; rows that do not (odd offsets of 16-bit
// types) are loaded and stored.
template <typename IO, int ROWS, int COLS, int NT, bool WIDE>
__device__ __forceinline__ void fill_tile(IO* dst, const IO* src, long long stride, int rows, int cols, bool words) {
    constexpr int E = (int)sizeof(IO);
    constexpr int BYTES = !WIDE ? 4 : COLS * E >= 16 ? 16 : COLS * E;
    constexpr int PER = BYTES / E, CPR = COLS / PER;
    if (WIDE || words) {
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * CPR; i += NT) {
            const int t = i / CPR, c = i % CPR * PER;
            int n = t < rows ? (cols - c) * E : 0;
            n = n < 0 ? 0 : n > BYTES ? BYTES : n;
            copy_async<BYTES>(dst + t * COLS + c, n ? src + t * stride + c : src, n);
        }
    } else {
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * COLS; i += NT) {
            const int t = i / COLS, c = i % COLS;
            dst[i] = t < rows && c < cols ? src[t * stride + c] : from_f<IO>(0.0f);
        }
    }
}

// The same for rows on 16-byte boundaries, for all tiles of a run: a thread has the same K pieces of
// every tile, so their addresses are formed once.  A block adds its tiles one after another; their
// pieces are dealt to the threads in that order.
template <typename IO, int ROWS, int NT, int K>
struct TilePieces {
    const char* src[K];
    long long step[K];                  // bytes from tile to tile
    unsigned dst[K];                    // byte in the stage
    int t[K], n[K];                     // step in the tile, bytes (0: no such piece)
    int next;                           // pieces dealt so far

    __device__ __forceinline__ void clear() {
        next = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) n[k] = -1;
    }
    template <int COLS> static constexpr int kBytes = COLS * (int)sizeof(IO) >= 16 ? 16 : 8;
    template <int COLS> static constexpr int kPieces = ROWS * (COLS * (int)sizeof(IO) / kBytes<COLS>);

    // the tile of COLS elements a row that lies `at` bytes into the stage
    template <int COLS>
    __device__ __forceinline__ void add(const void* base, const IO* from, long long stride, int cols) {
        constexpr int B = kBytes<COLS>, CPR = COLS * (int)sizeof(IO) / B;
        const unsigned at = smem_u32(base);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = k * NT + (int)threadIdx.x - next;
            if (i >= 0 && i < ROWS * CPR) {
                const int row = i / CPR, c = i % CPR * (B / (int)sizeof(IO));
                const int left = (cols - c) * (int)sizeof(IO);
                t[k] = row;
                n[k] = left < 0 ? 0 : left > B ? B : left;
                dst[k] = at + (row * COLS + c) * (int)sizeof(IO);
                src[k] = reinterpret_cast<const char*>(n[k] ? from + row * stride + c : from);
                step[k] = ROWS * stride * (long long)sizeof(IO);
                if (B == 8) n[k] |= 1 << 8;
            }
        }
        next += ROWS * CPR;
    }
    // copies of the current tile to the stage `offset` bytes on, and on to the next tile
    template <bool EIGHTS>
    __device__ __forceinline__ void issue(unsigned offset, int rows) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (n[k] >= 0) {
                const int bytes = t[k] < rows ? n[k] & 255 : 0;
                if (EIGHTS && (n[k] >> 8))
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst[k] + offset), "l"(src[k]), "r"(bytes) : "memory");
                else
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst[k] + offset), "l"(src[k]), "r"(bytes) : "memory");
                src[k] += step[k];
            }
        }
    }
};

}  // namespace dfsnn
