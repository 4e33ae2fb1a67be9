// Values to 4-bit block-scaled operands (MXF4, NVF4) and back.
//
// For a block of B consecutive values along k (B = 32 for MXF4, 16 for NVF4), y = x 2^-e and
// a = max |y|:
//     MXF4  s = 2^(floor(log2 a) - 2), no less than 2^-127       (the OCP microscaling rule)
//     NVF4  s = E4M3(min(a / 6, 448))
//     code  = E2M1(y / s), round to nearest even, magnitudes over 6 become 6
// A block of zeros, or whose scale rounds to zero, has codes of zero; one that holds an infinity
// or a NaN has the NaN scale and codes of zero.  Rounding twice (x to codes of a rounded scale)
// is what the formats are: nothing else here rounds.  y / s is exact for MXF4 (a power of two);
// for NVF4 see scaledBy().
//
// Both directions are bound by HBM: 2 + 17/32 bytes per 16-bit value.  A block of 256 threads
// takes 128 rows x 128 columns, so that the scale tiles it makes (512 bytes each) leave whole.
#include "common.cuh"
#include "mx_format.cuh"
#include "rocwmma/rocwmma_block.hpp"

namespace b200wmma
{
    using rocwmma::block::grid_dependency_wait;
    using rocwmma::block::grid_launch_dependents;

    namespace
    {
        constexpr uint32_t TILE_K  = 128;
        constexpr uint32_t THREADS = 256;

        // Eight consecutive values of a row, those at and behind `left` read as zero.
        template <typename T, bool VEC>
        __device__ inline void load8(T const* p, uint32_t left, float (&v)[8])
        {
            if(VEC && left >= 8u)
            {
                constexpr int N = int(sizeof(T) * 8 / 16);
                uint4         raw[N];
#pragma unroll
                for(int i = 0; i < N; ++i)
                    raw[i] = reinterpret_cast<uint4 const*>(p)[i];
                T const* t = reinterpret_cast<T const*>(raw);
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    v[i] = toFloat(t[i]);
            }
            else
            {
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    v[i] = uint32_t(i) < left ? toFloat(p[i]) : 0.0f;
            }
        }

        // Largest |v| as bits: ordered like the values, a NaN above the infinity.
        __device__ inline uint32_t topBits(float v, uint32_t top)
        {
            return max(top, __float_as_uint(v) & 0x7fffffffu);
        }

        // The scale of a block whose largest magnitude has these bits.
        struct Scale
        {
            uint32_t byte;
            float    inverse; // MXF4: exactly 1 / s; NVF4: 1 / s rounded; 0: codes are zero
            float    value;
        };
        template <bool NV>
        __device__ inline Scale scaleOf(uint32_t top)
        {
            const bool fine = top < 0x7f800000u;
            Scale      s;
            if constexpr(NV)
            {
                const float want = fminf(__fdiv_rn(__uint_as_float(fine ? top : 0u), 6.0f), 448.0f);
                const uint32_t byte = toE4m3(want);
                s.value             = fromE4m3(byte);
                s.inverse           = byte != 0u ? __frcp_rn(s.value) : 0.0f;
                s.byte              = fine ? byte : 0x7fu;
            }
            else
            {
                const uint32_t e    = (fine ? top : 0u) >> 23;
                const uint32_t byte = e > 2u ? e - 2u : 0u;
                s.value             = fromE8m0(byte);
                s.inverse           = fine ? __uint_as_float((254u - byte) << 23) : 0.0f;
                s.byte              = fine ? byte : 255u;
            }
            return s;
        }

        // y / s, exact as far as the rounding to E2M1 can see.  For NVF4 the borders between two
        // codes are multiples m s of a 4-bit s by a 3-bit m: at most seven significant bits.  A
        // quotient from 16-bit values (at most eleven bits) is on a border or at least 2^-11 of
        // its size away from it, so y * (1 / s), which is off by less than 2^-22, is rounded to
        // 14 bits: what lay on a border is there again, and nothing else gets there.  For 32-bit
        // values the division is rounded correctly, which keeps the order to every border.
        template <typename T, bool NV>
        __device__ inline float scaledBy(float y, Scale const& s)
        {
            if constexpr(!NV)
                return y * s.inverse;
            else if constexpr(sizeof(T) == 2)
            {
                const uint32_t q = __float_as_uint(y * s.inverse);
                return __uint_as_float((q + 0x200u) & ~0x3ffu);
            }
            else
                return s.inverse != 0.0f ? __fdiv_rn(y, s.value) : 0.0f;
        }

        // Inputs in which a NaN may meet an inverse of zero would make a NaN, whose code is not
        // zero; codes of such blocks are cleared as words.
        template <typename T, bool NV>
        __device__ inline uint32_t codes8(float const (&y)[8], Scale const& s)
        {
            float v[8];
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[i] = scaledBy<T, NV>(y[i], s);
            const uint32_t c = e2m1x8(v);
            return s.inverse != 0.0f ? c : 0u;
        }

        __device__ inline uint32_t scaleOffset(uint32_t row, uint32_t block)
        {
            return (block / 4u) * MX_TILE_BYTES + (row % 32u) * 16u + (row / 32u % 4u) * 4u
                   + block % 4u;
        }

        struct QuantizeParams
        {
            void const* x;
            uint8_t*    codes;
            uint8_t*    scales;
            uint64_t    ldq; // bytes
            uint64_t    ldx; // elements
            uint32_t    rows, k, groups, tilesK;
            float       factor; // 2^-exponent
        };

        // The scale tiles of one 128 x 128 tile, from shared memory, whole.
        template <bool NV>
        __device__ inline void storeScales(QuantizeParams const& p, uint8_t const* scales,
                                           uint32_t tileRow, uint32_t tileK)
        {
            constexpr uint32_t GROUPS = TILE_K / (4u * mxBlock(NV));
            const uint32_t     at     = threadIdx.x * 16u;
            const uint32_t     group  = tileK * GROUPS + at / MX_TILE_BYTES;
            if(at < GROUPS * MX_TILE_BYTES && group < p.groups)
                *reinterpret_cast<uint4*>(p.scales + (uint64_t(tileRow) * p.groups + group) * MX_TILE_BYTES
                                          + at % MX_TILE_BYTES)
                    = *reinterpret_cast<uint4 const*>(scales + at);
        }

        // x row-major: k is contiguous.  Sixteen threads read 128 values of a row, eight each;
        // a block's largest magnitude comes from its two (NVF4) or four (MXF4) threads.
        template <typename T, bool NV, bool VEC>
        __global__ void __launch_bounds__(THREADS) quantizeRowsKernel(const QuantizeParams p)
        {
            constexpr uint32_t GROUPS = TILE_K / (4u * mxBlock(NV));
            constexpr int      STEPS  = 128 / (THREADS / 16);
            __shared__ alignas(16) uint8_t scales[GROUPS * MX_TILE_BYTES];
            const uint32_t tileRow = blockIdx.x / p.tilesK, tileK = blockIdx.x % p.tilesK;
            const uint32_t col = threadIdx.x % 16u * 8u, rowIn = threadIdx.x / 16u;
            const uint32_t k0 = tileK * TILE_K + col;
            const uint32_t left = k0 < p.k ? p.k - k0 : 0u;
            grid_dependency_wait();
            grid_launch_dependents();
#pragma unroll
            for(int half = 0; half < 2; ++half)
            {
                float y[STEPS / 2][8];
#pragma unroll
                for(int i = 0; i < STEPS / 2; ++i)
                {
                    const uint64_t row = uint64_t(tileRow) * 128u + (half * (STEPS / 2) + i) * 16u + rowIn;
                    load8<T, VEC>(static_cast<T const*>(p.x) + row * p.ldx + k0, row < p.rows ? left : 0u, y[i]);
                }
#pragma unroll
                for(int i = 0; i < STEPS / 2; ++i)
                {
                    const uint32_t r   = (half * (STEPS / 2) + i) * 16u + rowIn;
                    const uint64_t row = uint64_t(tileRow) * 128u + r;
                    uint32_t       top = 0;
#pragma unroll
                    for(int j = 0; j < 8; ++j)
                    {
                        y[i][j] *= p.factor;
                        top = topBits(y[i][j], top);
                    }
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    if constexpr(!NV)
                        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const Scale    s    = scaleOf<NV>(top);
                    const uint32_t code = codes8<T, NV>(y[i], s);
                    if(col % mxBlock(NV) == 0u)
                        scales[scaleOffset(r, col / mxBlock(NV))] = uint8_t(s.byte);
                    if(row < p.rows && k0 / 2u < mxPitch(p.k))
                        *reinterpret_cast<uint32_t*>(p.codes + row * p.ldq + k0 / 2u) = code;
                }
            }
            __syncthreads();
            storeScales<NV>(p, scales, tileRow, tileK);
        }

        // x column-major: the rows are contiguous.  A thread takes two neighbouring rows and 32
        // values of k of each, so that a warp reads 64 consecutive values at a time and no
        // maximum crosses a thread; the codes pass through shared memory to leave as rows.
        template <typename T, bool NV, bool VEC>
        __global__ void __launch_bounds__(THREADS) quantizeColumnsKernel(const QuantizeParams p)
        {
            constexpr uint32_t GROUPS = TILE_K / (4u * mxBlock(NV));
            constexpr int      B      = int(mxBlock(NV));
            constexpr uint32_t PITCH  = 80; // of a staged row: 64 bytes of codes, 16 of padding
            __shared__ alignas(16) uint8_t scales[GROUPS * MX_TILE_BYTES];
            __shared__ alignas(16) uint8_t staged[128 * PITCH];
            const uint32_t tileRow = blockIdx.x / p.tilesK, tileK = blockIdx.x % p.tilesK;
            const uint32_t r = threadIdx.x % 64u * 2u, kIn = threadIdx.x / 64u * 32u;
            const uint64_t row = uint64_t(tileRow) * 128u + r;
            const uint32_t k0  = tileK * TILE_K + kIn;
            grid_dependency_wait();
            grid_launch_dependents();
            T        v[32][2];
            T const* x = static_cast<T const*>(p.x) + row;
#pragma unroll
            for(int i = 0; i < 32; ++i)
            {
                const bool in = k0 < p.k && uint32_t(i) < p.k - k0;
                T const*   at = x + (uint64_t(k0) + uint32_t(i)) * p.ldx;
                if constexpr(VEC)
                {
                    using Pair = typename std::conditional<sizeof(T) == 2, uint32_t, uint2>::type;
                    Pair w{};
                    if(in && row + 1u < p.rows)
                        w = *reinterpret_cast<Pair const*>(at);
                    else if(in && row < p.rows)
                    {
                        const T one[2] = {at[0], T(0.0f)};
                        w              = *reinterpret_cast<Pair const*>(one);
                    }
                    const T* pair = reinterpret_cast<T const*>(&w);
                    v[i][0]       = pair[0];
                    v[i][1]       = pair[1];
                }
                else
                {
                    v[i][0] = in && row < p.rows ? at[0] : T(0.0f);
                    v[i][1] = in && row + 1u < p.rows ? at[1] : T(0.0f);
                }
            }
#pragma unroll
            for(int j = 0; j < 2; ++j)
            {
                uint32_t words[4];
#pragma unroll
                for(int b = 0; b < 32 / B; ++b)
                {
                    uint32_t top = 0;
#pragma unroll
                    for(int i = 0; i < B; ++i)
                        top = topBits(toFloat(v[b * B + i][j]) * p.factor, top);
                    const Scale s = scaleOf<NV>(top);
#pragma unroll
                    for(int w = 0; w < B / 8; ++w)
                    {
                        float y[8];
#pragma unroll
                        for(int i = 0; i < 8; ++i)
                            y[i] = toFloat(v[b * B + w * 8 + i][j]) * p.factor;
                        words[b * (B / 8) + w] = codes8<T, NV>(y, s);
                    }
                    scales[scaleOffset(r + j, kIn / B + b)] = uint8_t(s.byte);
                }
                *reinterpret_cast<uint4*>(staged + (r + j) * PITCH + kIn / 2u)
                    = make_uint4(words[0], words[1], words[2], words[3]);
            }
            __syncthreads();
            storeScales<NV>(p, scales, tileRow, tileK);
            // four threads a row
            const uint64_t pitch = mxPitch(p.k);
            for(uint32_t i = threadIdx.x; i < 128u * 4u; i += THREADS)
            {
                const uint32_t rr = i / 4u;
                const uint64_t at = uint64_t(tileK) * (TILE_K / 2) + i % 4u * 16u;
                const uint64_t out = uint64_t(tileRow) * 128u + rr;
                if(out < p.rows && at < pitch)
                    *reinterpret_cast<uint4*>(p.codes + out * p.ldq + at)
                        = *reinterpret_cast<uint4 const*>(staged + rr * PITCH + i % 4u * 16u);
            }
        }

        struct DequantizeParams
        {
            uint8_t const* codes;
            uint8_t const* scales;
            void*          out;
            uint64_t       ldq; // bytes
            uint64_t       ldo; // elements
            uint32_t       rows, k, groups, tilesK;
            float          factor; // 2^exponent
        };

        template <typename T, bool NV, bool VEC>
        __global__ void __launch_bounds__(THREADS) dequantizeKernel(const DequantizeParams p)
        {
            constexpr int  STEPS   = 128 / (THREADS / 16);
            const uint32_t tileRow = blockIdx.x / p.tilesK, tileK = blockIdx.x % p.tilesK;
            const uint32_t k0 = tileK * TILE_K + threadIdx.x % 16u * 8u, rowIn = threadIdx.x / 16u;
            grid_dependency_wait();
            grid_launch_dependents();
            if(k0 >= p.k)
                return;
            uint32_t word[STEPS], byte[STEPS];
#pragma unroll
            for(int i = 0; i < STEPS; ++i)
            {
                const uint32_t r   = i * 16u + rowIn;
                const uint64_t row = uint64_t(tileRow) * 128u + r;
                word[i] = byte[i] = 0;
                if(row < p.rows)
                {
                    word[i] = *reinterpret_cast<uint32_t const*>(p.codes + row * p.ldq + k0 / 2u);
                    byte[i] = p.scales[uint64_t(tileRow) * p.groups * MX_TILE_BYTES
                                       + uint64_t(k0 / mxBlock(NV) / 4u) * MX_TILE_BYTES
                                       + scaleOffset(r, k0 / mxBlock(NV) % 4u)];
                }
            }
#pragma unroll
            for(int i = 0; i < STEPS; ++i)
            {
                const uint64_t row = uint64_t(tileRow) * 128u + i * 16u + rowIn;
                if(row >= p.rows)
                    continue;
                // code * s is exact (three bits times at most four); so is the power of two,
                // short of the subnormals
                const float s = NV ? fromE4m3(byte[i]) : fromE8m0(byte[i]);
                float       v[8];
                e2m1x8ToFloat(word[i], v);
                alignas(16) T out[8];
#pragma unroll
                for(int j = 0; j < 8; ++j)
                    out[j] = fromFloat<T>(v[j] * s * p.factor);
                T* at = static_cast<T*>(p.out) + row * p.ldo + k0;
                if(VEC && k0 + 8u <= p.k)
                {
#pragma unroll
                    for(int j = 0; j < int(sizeof(T) * 8 / 16); ++j)
                        reinterpret_cast<uint4*>(at)[j] = reinterpret_cast<uint4 const*>(out)[j];
                }
                else
                {
#pragma unroll
                    for(int j = 0; j < 8; ++j)
                        if(k0 + j < p.k)
                            at[j] = out[j];
                }
            }
        }

        bool aligned(void const* p, uint64_t bytes)
        {
            return reinterpret_cast<uintptr_t>(p) % bytes == 0;
        }

        template <typename T>
        int quantize(bool nv, bool columns, QuantizeParams const& p, uint32_t blocks, cudaStream_t stream)
        {
            // Wide loads where every row (or pair of rows) starts on their boundary.
            const uint64_t width = columns ? 2 * sizeof(T) : 16;
            const bool     vec   = aligned(p.x, width) && p.ldx * sizeof(T) % width == 0;
            auto launch = [&](auto kernel) {
                return cudaToStatus(launchOverlapped(kernel, dim3(blocks), dim3(THREADS), 0, stream, p));
            };
            if(columns)
                return nv ? (vec ? launch(quantizeColumnsKernel<T, true, true>) : launch(quantizeColumnsKernel<T, true, false>))
                          : (vec ? launch(quantizeColumnsKernel<T, false, true>) : launch(quantizeColumnsKernel<T, false, false>));
            return nv ? (vec ? launch(quantizeRowsKernel<T, true, true>) : launch(quantizeRowsKernel<T, true, false>))
                      : (vec ? launch(quantizeRowsKernel<T, false, true>) : launch(quantizeRowsKernel<T, false, false>));
        }

        template <typename T>
        int dequantize(bool nv, DequantizeParams const& p, uint32_t blocks, cudaStream_t stream)
        {
            const bool vec = aligned(p.out, 16) && p.ldo * sizeof(T) % 16 == 0;
            auto launch = [&](auto kernel) {
                return cudaToStatus(launchOverlapped(kernel, dim3(blocks), dim3(THREADS), 0, stream, p));
            };
            return nv ? (vec ? launch(dequantizeKernel<T, true, true>) : launch(dequantizeKernel<T, true, false>))
                      : (vec ? launch(dequantizeKernel<T, false, true>) : launch(dequantizeKernel<T, false, false>));
        }

        // What both directions check; OK or a status.
        int checkOperand(int fmt, int dtype, uint32_t rows, uint32_t k, void const* values,
                         uint64_t ld, uint64_t span, int exponent, void const* codes, uint64_t ldq,
                         void const* scales, uint64_t* blocks)
        {
            if(!values || !codes || !scales || rows == 0 || k == 0 || ld < span || ldq < mxPitch(k)
               || exponent < -64 || exponent > 64)
                return B200WMMA_ERR_INVALID_ARG;
            if(!mxFormat(fmt) || (dtype != B200WMMA_F16 && dtype != B200WMMA_BF16 && dtype != B200WMMA_F32))
                return B200WMMA_ERR_UNSUPPORTED;
            if(!aligned(codes, 16) || !aligned(scales, 16) || ldq % 16 || !aligned(values, dtypeSize(dtype)))
                return B200WMMA_ERR_ALIGNMENT;
            *blocks = uint64_t(mxRowTiles(rows)) * ((uint64_t(k) + TILE_K - 1) / TILE_K);
            if(*blocks > 0x7fffffffull)
                return B200WMMA_ERR_TOO_LARGE;
            return B200WMMA_OK;
        }
    } // namespace
} // namespace b200wmma

using namespace b200wmma;

extern "C" {

uint64_t b200wmma_mx_pitch(uint32_t k)
{
    return mxPitch(k);
}

uint64_t b200wmma_mx_scale_bytes(int fmt, uint32_t rows, uint32_t k)
{
    if(!mxFormat(fmt))
        return 0;
    return uint64_t(mxRowTiles(rows)) * mxGroups(fmt == B200WMMA_NVF4, k) * MX_TILE_BYTES;
}

int b200wmma_mx_quantize(int fmt, int in_dtype, uint32_t rows, uint32_t k, const void* x,
                         uint64_t ldx, int layout, int exponent, void* codes, uint64_t ldq,
                         void* scales, void* stream)
{
    const bool columns = layout == B200WMMA_COL_MAJOR;
    if(layout != B200WMMA_ROW_MAJOR && !columns)
        return B200WMMA_ERR_INVALID_ARG;
    uint64_t  blocks = 0;
    const int rc = checkOperand(fmt, in_dtype, rows, k, x, ldx, columns ? rows : k, exponent, codes,
                                ldq, scales, &blocks);
    if(rc != B200WMMA_OK)
        return rc;
    const bool           nv = fmt == B200WMMA_NVF4;
    const QuantizeParams p{x, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), ldq, ldx,
                           rows, k, mxGroups(nv, k), uint32_t((uint64_t(k) + TILE_K - 1) / TILE_K),
                           ldexpf(1.0f, -exponent)};
    const cudaStream_t   s = static_cast<cudaStream_t>(stream);
    switch(in_dtype)
    {
    case B200WMMA_F16:
        return quantize<__half>(nv, columns, p, uint32_t(blocks), s);
    case B200WMMA_BF16:
        return quantize<__nv_bfloat16>(nv, columns, p, uint32_t(blocks), s);
    }
    return quantize<float>(nv, columns, p, uint32_t(blocks), s);
}

int b200wmma_mx_dequantize(int fmt, int out_dtype, uint32_t rows, uint32_t k, const void* codes,
                           uint64_t ldq, const void* scales, int exponent, void* out, uint64_t ldo,
                           void* stream)
{
    uint64_t  blocks = 0;
    const int rc = checkOperand(fmt, out_dtype, rows, k, out, ldo, k, exponent, codes, ldq, scales, &blocks);
    if(rc != B200WMMA_OK)
        return rc;
    const bool             nv = fmt == B200WMMA_NVF4;
    const DequantizeParams p{static_cast<uint8_t const*>(codes), static_cast<uint8_t const*>(scales),
                             out, ldq, ldo, rows, k, mxGroups(nv, k),
                             uint32_t((uint64_t(k) + TILE_K - 1) / TILE_K), ldexpf(1.0f, exponent)};
    const cudaStream_t     s = static_cast<cudaStream_t>(stream);
    switch(out_dtype)
    {
    case B200WMMA_F16:
        return dequantize<__half>(nv, p, uint32_t(blocks), s);
    case B200WMMA_BF16:
        return dequantize<__nv_bfloat16>(nv, p, uint32_t(blocks), s);
    }
    return dequantize<float>(nv, p, uint32_t(blocks), s);
}
}
