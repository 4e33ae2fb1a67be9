// The 4-bit block-scaled formats: element and scale encodings and the storage layout shared by
// the kernels that write (mx_quantize.cu) and read (mx_quantize.cu, mx_gemm.cu) them.
//
// An operand is `rows` x `k` values.  Codes: E2M1, two to a byte, the even column in the low
// four bits; a row takes ceil(k / 32) * 16 bytes (or a larger multiple of 16 the caller names),
// which is what the TMA needs of a row pitch.  Scales: one byte per block of 32 (MXF4, E8M0) or
// 16 (NVF4, E4M3) consecutive k, stored in tiles of 128 rows x 4 blocks = 512 bytes in the order
// [row tile][block group][row % 32][row / 32 % 4][block % 4]: exactly the 32 x 16-byte picture
// that tcgen05.cp spreads over tensor memory, so that the product copies tiles and never
// rearranges them.
#ifndef ROCWMMA_B200_CSRC_MX_FORMAT_CUH
#define ROCWMMA_B200_CSRC_MX_FORMAT_CUH

#include "rocwmma_b200.h"
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200wmma
{
    constexpr uint32_t MX_TILE_ROWS  = 128;
    constexpr uint32_t MX_TILE_BYTES = 512;

    inline bool mxFormat(int fmt)
    {
        return fmt == B200WMMA_MXF4 || fmt == B200WMMA_NVF4;
    }
    __host__ __device__ constexpr uint32_t mxBlock(bool nv)
    {
        return nv ? 16u : 32u;
    }
    __host__ __device__ inline uint64_t mxPitch(uint32_t k)
    {
        return (uint64_t(k) + 31u) / 32u * 16u;
    }
    __host__ __device__ inline uint32_t mxRowTiles(uint32_t rows)
    {
        return uint32_t((uint64_t(rows) + 127u) / 128u);
    }
    __host__ __device__ inline uint32_t mxGroups(bool nv, uint32_t k) // groups of four blocks
    {
        const uint32_t span = 4u * mxBlock(nv);
        return uint32_t((uint64_t(k) + span - 1u) / span);
    }

#ifdef __CUDACC__
    __device__ inline float toFloat(__half v)
    {
        return __half2float(v);
    }
    __device__ inline float toFloat(__nv_bfloat16 v)
    {
        return __bfloat162float(v);
    }
    __device__ inline float toFloat(float v)
    {
        return v;
    }
    template <typename T>
    __device__ inline T fromFloat(float v)
    {
        return T(v); // round to nearest even
    }

    // Eight values to eight codes, value i in bits 4 i..4 i + 3: nearest E2M1 value, ties to the
    // even code, magnitudes over 6 become 6.
    __device__ inline uint32_t e2m1x8(float const (&v)[8])
    {
        uint32_t r;
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
            "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
            : "=r"(r)
            : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]),
              "f"(v[7]));
        return r;
    }
    // ... and back.
    __device__ inline void e2m1x8ToFloat(uint32_t codes, float (&v)[8])
    {
        uint32_t h[4];
        asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
            "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
            "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
            : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
            : "r"(codes));
#pragma unroll
        for(int i = 0; i < 4; ++i)
        {
            const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
            v[2 * i]       = f.x;
            v[2 * i + 1]   = f.y;
        }
    }
    // E4M3, saturating at 448.
    __device__ inline uint32_t toE4m3(float v)
    {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
        return r & 0xffu;
    }
    __device__ inline float fromE4m3(uint32_t byte)
    {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(byte)));
        return __half2float(__ushort_as_half(uint16_t(h & 0xffffu)));
    }
    // E8M0: 2^(byte - 127); 255 is NaN.
    __device__ inline float fromE8m0(uint32_t byte)
    {
        return byte == 255u ? __uint_as_float(0x7fffffffu)
                            : __uint_as_float(byte == 0u ? 0x00400000u : byte << 23);
    }
#endif
} // namespace b200wmma
#endif
