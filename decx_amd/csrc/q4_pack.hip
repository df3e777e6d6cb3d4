// From a matrix to 4 bits and back (layout: gemm_q4.hpp).
//
//   without zero points   scale = max|w| / 7,          code = clamp(rint(w / scale), -8, 7) + 8
//   with zero points      lo = min(0, min w), hi = max(0, max w), scale = (hi - lo) / 15,
//                         zero = clamp(rint(-lo / scale), 0, 15),  code = clamp(rint(w / scale) + zero, 0, 15)
//
// over the group's columns; scale is computed in fp32 and held in fp16, and what follows uses the held one.  Halves round to
// even, and a quotient next to a half is decided exactly, so that a code never depends on how a quotient was rounded.
// A wavefront makes one tile: whole rows of it turned around in LDS, so that a lane holds 8 adjacent columns of its row four times,
// the extremes of a group met over the row's 4 lanes, and the tile stored 16 bytes per lane, 1 KB in a row.
// Bound: 4096 x 4096 fp16 to 4 bits 12-15 us traced, 42 MB at 2.9-3.4 TB/s: a wavefront's one chain of load, extremes, codes and store (it
// waits 59 % of its time; the vector pipe, about ten instructions a weight, is half busy).  5003 x 7001 fp32 in groups of 32 with
// zero points 43.5 us, 3.9 TB/s.  Back to fp32: 13.2 and 30.1 us, HBM (5.7 and 5.4 TB/s).
#include "gemm_q4.hpp"

namespace decx_hip {

namespace {

// eight adjacent weights as they lie in memory
struct EightF32 { floatx4 a, b; };
template <typename T> struct Eight { typedef halfx8 type; };
template <> struct Eight<float> { typedef EightF32 type; };
__device__ __forceinline__ float element(const halfx8& r, int e) { return (float)r[e]; }
__device__ __forceinline__ float element(const EightF32& r, int e) { return e < 4 ? r.a[e] : r.b[e - 4]; }

// lo and hi (ZEROS only) and the bits of the largest magnitude so far, as fp32
template <bool ZEROS> __device__ __forceinline__ void extremes(const halfx8& r, float& lo, float& hi, uint32_t& top)
{
    // two at a time: magnitudes as whole numbers
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const uintx4 w = __builtin_bit_cast(uintx4, r);
    u16x2 m = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
    const uint16_t one = m[0] > m[1] ? m[0] : m[1];
    const uint32_t bits = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, one));      // (NaN stays NaN, infinity infinity)
    top = bits > top ? bits : top;
    if (ZEROS) {
#pragma unroll
        for (int e = 0; e < 8; ++e) { lo = __builtin_fminf(lo, (float)r[e]); hi = __builtin_fmaxf(hi, (float)r[e]); }
    }
}
template <bool ZEROS> __device__ __forceinline__ void extremes(const EightF32& r, float& lo, float& hi, uint32_t& top)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = element(r, e);
        const uint32_t bits = __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
        top = bits > top ? bits : top;
        if (ZEROS) { lo = __builtin_fminf(lo, x); hi = __builtin_fmaxf(hi, x); }
    }
}
// rint(w / s) by comparison with the half s (m + 1/2) next to the quotient, m = floor(v), v the quotient in fp32: the half is
// exact in fp32 (11 bits times 6, for quotients that a code can hold), so this is too, ties to even included.
__device__ __forceinline__ float rint_exactly(float w, float s, float v)
{
    const float m = __builtin_floorf(v), half = s * (m + 0.5f);
    const float even = 2.f * __builtin_rintf(0.5f * m + 0.25f);         // of m and m + 1 the even one
    return w > half ? m + 1.f : (w < half ? m : even);
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
    // rows of the tile in LDS: 16-byte chunk c of row r in slot c ^ r, so that 16 rows of a chunk cover all banks
    constexpr int E = 16 / sizeof(T), CPR = kQ4TileCols / E, AT_ONCE = 64 / CPR;
    __shared__ __attribute__((aligned(1024))) unsigned char all[PACK_WAVES][16 * CPR * 16];
    unsigned char* const lds = all[threadIdx.x >> 6];
    const uint32_t row0 = (uint32_t)(tile / k_tiles) * kQ4TileRows, col0 = (uint32_t)(tile % k_tiles) * kQ4TileCols;
    const int load_row = lane / CPR, chunk = lane % CPR;
    uintx4 loaded[CPR / 4];
    if (row0 + 16 <= N && col0 + kQ4TileCols <= K) {
#pragma unroll
        for (int c = 0; c < CPR / 4; ++c) __builtin_memcpy(&loaded[c], W + (size_t)(row0 + load_row + c * AT_ONCE) * ldw + col0 + chunk * E, 16);
    } else {
#pragma unroll
        for (int c = 0; c < CPR / 4; ++c) {
            const uint32_t n = row0 + load_row + c * AT_ONCE;
            loaded[c] = n < N ? load_end(W + (size_t)n * ldw, col0 + chunk * E, K) : uintx4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for (int c = 0; c < CPR / 4; ++c) *(uintx4*)(lds + ((load_row + c * AT_ONCE) * CPR + (chunk ^ (load_row + c * AT_ONCE))) * 16) = loaded[c];
    wavefront_order();
    typename Eight<T>::type raw[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uintx4 v[8 / E];
#pragma unroll
        for (int h = 0; h < 8 / E; ++h) v[h] = *(const uintx4*)(lds + (r * CPR + (((j * 4 + kg) * (8 / E) + h) ^ r)) * 16);
        raw[j] = __builtin_bit_cast(typename Eight<T>::type, v);
    }
    constexpr int STEPS = 4 / GPB;
    uintx4 out;
#pragma unroll
    for (int q = 0; q < GPB; ++q) {
        // The extremes, and whether everything is finite (the largest magnitude's bits: a NaN's are above all others').
        float lo = 0.f, hi = 0.f;
        uint32_t top = 0;
#pragma unroll
        for (int j = q * STEPS; j < (q + 1) * STEPS; ++j) extremes<ZEROS>(raw[j], lo, hi, top);
#pragma unroll
        for (int off = 16; off <= 32; off <<= 1) {
            if (ZEROS) {
                const float l = __shfl_xor(lo, off, 64), h = __shfl_xor(hi, off, 64);
                lo = l < lo ? l : lo;
                hi = h > hi ? h : hi;
            }
            const uint32_t b = __shfl_xor(top, off, 64);
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
            z = rint_exactly(-lo, s, -lo * inverse);
            z = z > 15.f ? 15.f : z;
        }
        const float most = 15.f - z, least = -z;
        const uint32_t eight_z = (uint32_t)(int)z * 0x11111111u;
#pragma unroll
        for (int j = q * STEPS; j < (q + 1) * STEPS; ++j) {
            // v is off by less than 17 * 2^-23; only where that is enough to cross a half is the exact form asked
            float v[8], c[8], near = 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = element(raw[j], e) * inverse;
                c[e] = __builtin_rintf(v[e]);
                near = __builtin_fminf(near, __builtin_fabsf(__builtin_fabsf(v[e] - c[e]) - 0.5f));
            }
            if (near < 4e-6f) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (__builtin_fabsf(v[e]) < 17.f) c[e] = rint_exactly(element(raw[j], e), s, v[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = __builtin_amdgcn_fmed3f(c[e], least, most);
            // the word's nibbles hold columns 0, 2, 4, 6, 1, 3, 5, 7: four to a sum in fp32, which holds them exactly
            const auto four = [&](int e) { return (int)__builtin_fmaf(c[e + 6], 4096.f, __builtin_fmaf(c[e + 4], 256.f, __builtin_fmaf(c[e + 2], 16.f, c[e]))); };
            const uint32_t word = (uint32_t)four(0) + ((uint32_t)four(1) << 16) + eight_z;     // (borrows of negative ones are made good by the zero points)
            out[j] = some ? word : eight_z;
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
    constexpr int E = 16 / sizeof(T), CPR = kQ4TileCols / E, AT_ONCE = 64 / CPR;
    __shared__ __attribute__((aligned(1024))) unsigned char all[PACK_WAVES][16 * CPR * 16];
    unsigned char* const lds = all[threadIdx.x >> 6];
    const uintx4 w = *(const uintx4*)(codes + tile * kQ4TileBytes + lane * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const size_t at = (tile * 16 + r) * GPB + j * GPB / 4;
        const float s = (float)scales[at];
        const int z = zeros ? zeros[at] : 8;
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)((float)((int)((w[j] >> (4 * (e / 2 + 4 * (e % 2)))) & 15u) - z) * s);     // 5 bits by 11: exact in fp32
#pragma unroll
        for (int h = 0; h < 8 / E; ++h) __builtin_memcpy(lds + (r * CPR + (((j * 4 + kg) * (8 / E) + h) ^ r)) * 16, v + h * E, 16);
    }
    wavefront_order();
    const uint32_t row0 = (uint32_t)(tile / k_tiles) * kQ4TileRows, col0 = (uint32_t)(tile % k_tiles) * kQ4TileCols;
    const int store_row = lane / CPR, chunk = lane % CPR;
    const uint32_t k = col0 + chunk * E;
#pragma unroll
    for (int c = 0; c < CPR / 4; ++c) {
        const uint32_t n = row0 + store_row + c * AT_ONCE;
        if (n >= N || k >= K) continue;
        const uintx4 v = *(const uintx4*)(lds + ((store_row + c * AT_ONCE) * CPR + (chunk ^ (store_row + c * AT_ONCE))) * 16);
        T* p = W + (size_t)n * ldw + k;
        if (k + E <= K) {
            __builtin_memcpy(p, &v, 16);
        } else {
            T one[E];
            __builtin_memcpy(one, &v, 16);
#pragma unroll
            for (int e = 0; e < E; ++e) if (k + e < K) p[e] = one[e];
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
