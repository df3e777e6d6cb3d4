// Shared declarations of the 4-bit layer: products with weights held in 4 bits, the step that makes such weights, and
// the root-mean-square norm in front of them.
#pragma once
#include "gemm_common.hpp"

namespace decx_hip {

// Where a 4-bit matrix of N rows x K columns keeps its parts.  Tiles of 16 rows x 128 columns, 1024 bytes each,
// [row tile][column tile]: one 16-byte piece per lane of a wavefront in the order the matrix instruction wants its
// operand, so that a wavefront's load of a tile is 1 KB in a row and no code changes lanes on its way.  Lane 16 kg + r
// holds row r; word j of its piece the columns 32 j + 8 kg + 0..7, in nibbles 0, 4, 1, 5, 2, 6, 3, 7: masking the word
// with 0x000f000f (0x00f000f0, ...) then gives two adjacent columns in two halves.  Scales and zero points lie
// [row tile][column tile][row][group of the tile].
constexpr uint32_t kQ4TileRows = 16, kQ4TileCols = 128, kQ4TileBytes = 1024;

struct GemmQ4Args {
    const void* X;               // fp16 or int8, M x K
    const float* x_scales;       // int8: a factor per row of X
    const unsigned char* codes;
    const _Float16* scales;
    const unsigned char* zeros;  // or null: 8 everywhere
    const void* C;               // of Y's type, or null; ldc = 0: one row for all
    void* Y;                     // fp16, or fp32 with y_f32
    uint32_t M, N, K;
    uint32_t ldx, ldc, ldy;
    float alpha, beta;
    uint32_t y_f32;
    uint32_t k_tiles, n_tiles;   // tiles of W along K and N
    uint32_t quads_ok;           // 1: C and Y may be read and written 4 elements at a time
    uint32_t tiles_m, tiles_n;   // block tiles
    uint32_t splits;             // ranges of K with workgroups of their own, split_tiles tiles of W each (1: none)
    uint32_t split_tiles;
    uint32_t partial_ld;         // their sums: [range][row][partial_ld], a multiple of 4
    float* partial;
};

enum GemmQ4Kernel : int {
    Q4_ROWS_16_NARROW, Q4_ROWS_16, Q4_ROWS_16_WIDE, Q4_ROWS_32_NARROW, Q4_ROWS_32, Q4_ROWS_64_NARROW, Q4_ROWS_64,
    Q4_TILES_64x128, Q4_TILES_64x256, Q4_TILES_128x384, Q4_KERNEL_COUNT,
};
struct GemmQ4Plan { int kernel; uint32_t splits, split_tiles; };
GemmQ4Plan plan_gemm_q4(bool i8, uint32_t group, uint32_t M, uint32_t N, uint32_t K, size_t workspace_bytes);
size_t gemm_q4_workspace(bool i8, uint32_t group, uint32_t M, uint32_t N, uint32_t K);
uint32_t gemm_q4_rows_a_launch(int kernel, uint32_t M, uint32_t N);
// whether `plan` is one that plan_gemm_q4 could give for such a product and workspace
bool gemm_q4_plan_ok(const GemmQ4Plan& plan, uint32_t M, uint32_t N, uint32_t K, size_t workspace_bytes);
// fills in the fields of a split; the workspace is 16-byte aligned and has room for the plan's sums
int launch_gemm_q4(bool i8, uint32_t group, const GemmQ4Args& args, const GemmQ4Plan& plan, void* workspace, hipStream_t stream);

int launch_q4_quantize(bool f16, const void* W, uint32_t N, uint32_t K, uint32_t ldw, uint32_t group, void* codes, void* scales,
                       void* zeros, hipStream_t stream);
int launch_q4_dequantize(bool f16, const void* codes, const void* scales, const void* zeros, void* W, uint32_t N, uint32_t K,
                         uint32_t ldw, uint32_t group, hipStream_t stream);

struct RmsNormArgs {
    const void* x;
    const void* residual;        // or null
    const void* weight;
    void* sum;                   // x + residual, or null
    void* y;                     // rows' type, or int8 with y_scales
    float* y_scales;
    uint32_t rows, cols, ldx, ldr, lds, ldy;
    float eps;
};
int launch_rmsnorm(bool f16, const RmsNormArgs& args, hipStream_t stream);

// 16 bytes of a row from column k on, zero from column K on (for the last columns; K >= 1): the 16 bytes that end at K,
// shifted down, so that one load does and nothing behind the row is read.
template <typename T> __device__ __forceinline__ uintx4 load_end(const T* row, uint32_t k, uint32_t K)
{
    constexpr uint32_t E = 16 / sizeof(T);
    uint64_t low = 0, high = 0;
    if (k < K && K >= E) {
        const uint32_t first = k + E <= K ? k : K - E, shift = (k - first) * 8 * sizeof(T);
        uintx4 v;
        __builtin_memcpy(&v, row + first, 16);
        low = (uint64_t)v[1] << 32 | v[0];
        high = (uint64_t)v[3] << 32 | v[2];
        if (shift >= 64) { low = high >> (shift - 64); high = 0; }
        else { low = low >> shift | high << 1 << (63 - shift); high >>= shift; }
    } else if (k < K) {
#pragma unroll 1
        for (uint32_t e = 0; k + e < K; ++e) {             // (rows shorter than that)
            typename std::conditional<sizeof(T) == 1, uint8_t, typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type>::type bits;
            __builtin_memcpy(&bits, row + k + e, sizeof(T));
            const uint32_t at = e * 8 * sizeof(T);
            if (at < 64) low |= (uint64_t)bits << at; else high |= (uint64_t)bits << (at - 64);
        }
    }
    return uintx4{(uint32_t)low, (uint32_t)(low >> 32), (uint32_t)high, (uint32_t)(high >> 32)};
}

// orders a wavefront's accesses to LDS of its own, which no other wavefront waits for
__device__ __forceinline__ void wavefront_order()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

}  // namespace decx_hip
