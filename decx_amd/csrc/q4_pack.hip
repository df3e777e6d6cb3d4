// From a matrix to 4 bits and back (layout: gemm_q4.hpp).
//
//   without zero points   scale = max|w| / 7,          code = clamp(rint(w / scale), -8, 7) + 8
//   with zero points      lo = min(0, min w), hi = max(0, max w), scale = (hi - lo) / 15,
//                         zero = clamp(rint(-lo / scale), 0, 15),  code = clamp(rint(w / scale) + zero, 0, 15)
//
// over the group's columns; scale is computed in fp32 and held in fp16, and what follows uses the held one.  Halves round to
// even, and a quotient next to a half is decided in 64 bits, so that a code never depends on how a quotient was rounded.
// Bound: HBM (N K elements in, half a byte each out).  A wavefront makes one tile: a lane reads 8 adjacent columns of its row
// four times (a row's 4 lanes cover 64 or 128 bytes in a row), the extremes of a group meet over those 4 lanes, and the tile
// is stored 16 bytes per lane, 1 KB in a row.
#include "gemm_q4.hpp"

namespace decx_hip {

namespace {

typedef halfx8 halfx8_u __attribute__((aligned(2)));
typedef floatx4 floatx4_u __attribute__((aligned(4)));

__device__ __forceinline__ void load8(const _Float16* p, float (&v)[8])
{
    const halfx8 h = *(const halfx8_u*)p;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8])
{
    const floatx4 a = *(const floatx4_u*)p, b = *(const floatx4_u*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
}
__device__ __forceinline__ void store8(_Float16* p, const float (&v)[8])
{
    halfx8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (_Float16)v[e];
    *(halfx8_u*)p = h;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8])
{
    *(floatx4_u*)p = floatx4{v[0], v[1], v[2], v[3]};
    *(floatx4_u*)(p + 4) = floatx4{v[4], v[5], v[6], v[7]};
}

// rint(w / s) for |w / s| of at most a few tens; inverse = 1 / s in fp32.  The fp32 product is off by less than
// 16 * 2^-22; only a result that close to a half is asked of the division in 64 bits.
__device__ __forceinline__ float rint_quotient(float w, float s, float inverse)
{
    const float v = w * inverse, r = __builtin_rintf(v);
    if (__builtin_fabsf(__builtin_fabsf(v - r) - 0.5f) < 1e-4f) return (float)__builtin_rint((double)w / (double)s);
    return r;
}

}  // namespace

constexpr int PACK_WAVES = 4;

template <typename T, int GPB, bool ZEROS>
__global__ void __launch_bounds__(PACK_WAVES * 64)
q4_quantize_kernel(const T* __restrict__ W, uint32_t N, uint32_t K, uint32_t ldw, uint32_t k_tiles, uint64_t tiles, unsigned char* __restrict__ codes,
                   _Float16* __restrict__ scales, unsigned char* __restrict__ zeros)
{
    const uint64_t tile = (uint64_t)blockIdx.x * PACK_WAVES + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int lane = threadIdx.x & 63, r = lane & 15, kg = lane >> 4;
    const uint32_t n = (uint32_t)(tile / k_tiles) * kQ4TileRows + r, k0 = (uint32_t)(tile % k_tiles) * kQ4TileCols + 8 * kg;
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t k = k0 + 32 * j;
        const T* p = W + (size_t)n * ldw + k;
        if (n < N && k + 8 <= K) {
            load8(p, v[j]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = n < N && k + e < K ? (float)p[e] : 0.f;
        }
    }
    constexpr int STEPS = 4 / GPB;
    uintx4 out;
#pragma unroll
    for (int q = 0; q < GPB; ++q) {
        // The extremes, and whether everything is finite (the largest magnitude's bits: a NaN's are above all others').
        float lo = 0.f, hi = 0.f;
        uint32_t top = 0;
#pragma unroll
        for (int j = q * STEPS; j < (q + 1) * STEPS; ++j)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = v[j][e];
                lo = x < lo ? x : lo;
                hi = x > hi ? x : hi;
                const uint32_t bits = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
                top = bits > top ? bits : top;
            }
#pragma unroll
        for (int off = 16; off <= 32; off <<= 1) {
            const float l = __shfl_xor(lo, off, 64), h = __shfl_xor(hi, off, 64);
            const uint32_t b = __shfl_xor(top, off, 64);
            lo = l < lo ? l : lo;
            hi = h > hi ? h : hi;
            top = b > top ? b : top;
        }
        const bool finite = top < 0x7f800000u;
        float s = ZEROS ? (hi - lo) / 15.f : __builtin_bit_cast(float, top) / 7.f;
        s = s > 65504.f ? 65504.f : s;                     // what fp16 can hold
        const _Float16 held = finite ? (_Float16)s : __builtin_bit_cast(_Float16, (uint16_t)0x7e00);
        s = finite ? (float)held : 0.f;
        const bool some = s > 0.f;
        const float inverse = some ? 1.f / s : 0.f;        // (the smallest fp16 is 2^-24: its inverse is finite)
        float z = 8.f;
        if (ZEROS && some) {
            z = (float)__builtin_rint(-(double)lo / (double)s);
            z = z > 15.f ? 15.f : z;
        }
        const float most = 15.f - z, least = -z;
#pragma unroll
        for (int j = q * STEPS; j < (q + 1) * STEPS; ++j) {
            uint32_t word = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float c = 0.f;
                if (some) {
                    // a weight beyond the clamp's range by more than a step is clamped before it is divided
                    const float w = v[j][e], far = 17.f * s, in = w > far ? far : (w < -far ? -far : w);
                    c = rint_quotient(in, s, inverse);
                    c = c > most ? most : (c < least ? least : c);
                }
                word |= (uint32_t)(int)(c + z) << (4 * (e / 2 + 4 * (e % 2)));
            }
            out[j] = word;
        }
        if (kg == q % 4) {
            const size_t at = (tile * 16 + r) * GPB + q;
            scales[at] = held;
            if (ZEROS) zeros[at] = (unsigned char)z;
        }
    }
    *(uintx4*)(codes + tile * kQ4TileBytes + lane * 16) = out;
}

template <typename T, int GPB>
__global__ void __launch_bounds__(PACK_WAVES * 64)
q4_dequantize_kernel(const unsigned char* __restrict__ codes, const _Float16* __restrict__ scales, const unsigned char* __restrict__ zeros,
                     uint32_t N, uint32_t K, uint32_t ldw, uint32_t k_tiles, uint64_t tiles, T* __restrict__ W)
{
    const uint64_t tile = (uint64_t)blockIdx.x * PACK_WAVES + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int lane = threadIdx.x & 63, r = lane & 15, kg = lane >> 4;
    const uint32_t n = (uint32_t)(tile / k_tiles) * kQ4TileRows + r, k0 = (uint32_t)(tile % k_tiles) * kQ4TileCols + 8 * kg;
    if (n >= N) return;
    const uintx4 w = *(const uintx4*)(codes + tile * kQ4TileBytes + lane * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const size_t at = (tile * 16 + r) * GPB + j * GPB / 4;
        const float s = (float)scales[at];
        const int z = zeros ? zeros[at] : 8;
        const uint32_t k = k0 + 32 * j;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)((int)((w[j] >> (4 * (e / 2 + 4 * (e % 2)))) & 15u) - z) * s;     // 5 bits by 11: exact in fp32
        T* p = W + (size_t)n * ldw + k;
        if (k + 8 <= K) {
            store8(p, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) if (k + e < K) p[e] = (T)v[e];
        }
    }
}

namespace {

template <typename T, int GPB>
void quantize_as(const void* W, uint32_t N, uint32_t K, uint32_t ldw, void* codes, void* scales, void* zeros, hipStream_t stream)
{
    const uint32_t kt = (K + kQ4TileCols - 1) / kQ4TileCols;
    const uint64_t tiles = (uint64_t)kt * ((N + kQ4TileRows - 1) / kQ4TileRows);
    const dim3 grid((unsigned)((tiles + PACK_WAVES - 1) / PACK_WAVES)), block(PACK_WAVES * 64);
    if (zeros)
        hipLaunchKernelGGL((q4_quantize_kernel<T, GPB, true>), grid, block, 0, stream, (const T*)W, N, K, ldw, kt, tiles, (unsigned char*)codes, (_Float16*)scales, (unsigned char*)zeros);
    else
        hipLaunchKernelGGL((q4_quantize_kernel<T, GPB, false>), grid, block, 0, stream, (const T*)W, N, K, ldw, kt, tiles, (unsigned char*)codes, (_Float16*)scales, (unsigned char*)nullptr);
}

template <typename T, int GPB>
void dequantize_as(const void* codes, const void* scales, const void* zeros, void* W, uint32_t N, uint32_t K, uint32_t ldw, hipStream_t stream)
{
    const uint32_t kt = (K + kQ4TileCols - 1) / kQ4TileCols;
    const uint64_t tiles = (uint64_t)kt * ((N + kQ4TileRows - 1) / kQ4TileRows);
    const dim3 grid((unsigned)((tiles + PACK_WAVES - 1) / PACK_WAVES)), block(PACK_WAVES * 64);
    hipLaunchKernelGGL((q4_dequantize_kernel<T, GPB>), grid, block, 0, stream, (const unsigned char*)codes, (const _Float16*)scales, (const unsigned char*)zeros, N, K, ldw, kt, tiles, (T*)W);
}

}  // namespace

// (the caller sees to it that the tiles fit a grid)
int launch_q4_quantize(bool f16, const void* W, uint32_t N, uint32_t K, uint32_t ldw, uint32_t group, void* codes, void* scales,
                       void* zeros, hipStream_t stream)
{
    const auto as = [&](auto gpb) {
        constexpr int GPB = decltype(gpb)::value;
        if (f16) quantize_as<_Float16, GPB>(W, N, K, ldw, codes, scales, zeros, stream);
        else quantize_as<float, GPB>(W, N, K, ldw, codes, scales, zeros, stream);
    };
    if (group == 128) as(std::integral_constant<int, 1>{});
    else if (group == 64) as(std::integral_constant<int, 2>{});
    else as(std::integral_constant<int, 4>{});
    return (int)hipGetLastError();
}

int launch_q4_dequantize(bool f16, const void* codes, const void* scales, const void* zeros, void* W, uint32_t N, uint32_t K,
                         uint32_t ldw, uint32_t group, hipStream_t stream)
{
    const auto as = [&](auto gpb) {
        constexpr int GPB = decltype(gpb)::value;
        if (f16) dequantize_as<_Float16, GPB>(codes, scales, zeros, W, N, K, ldw, stream);
        else dequantize_as<float, GPB>(codes, scales, zeros, W, N, K, ldw, stream);
    };
    if (group == 128) as(std::integral_constant<int, 1>{});
    else if (group == 64) as(std::integral_constant<int, 2>{});
    else as(std::integral_constant<int, 4>{});
    return (int)hipGetLastError();
}

}  // namespace decx_hip
