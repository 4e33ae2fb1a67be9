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
// Both directions are bound by HBM: 2 + 17/32 bytes per 16-bit value.
#include "common.cuh"
#include "mx_format.cuh"
#include "rocwmma/rocwmma_block.hpp"
#include <cstring>
#include <type_traits>

namespace b200wmma
{
    using rocwmma::block::grid_dependency_wait;
    using rocwmma::block::grid_launch_dependents;

    namespace
    {
        constexpr uint32_t TILE_K    = 128;
        constexpr uint32_t THREADS   = 256;
        constexpr uint32_t SLAB_ROWS = 32; // rows of a block: one 32-bit word of each scale tile row

        // Eight consecutive values of a row as they are stored.
        template <typename T>
        struct alignas(16) Raw8
        {
            T v[8];
        };
        template <typename T>
        __device__ inline Raw8<T> zero8()
        {
            Raw8<T> r;
#pragma unroll
            for(int i = 0; i < 8; ++i)
                r.v[i] = T(0.0f);
            return r;
        }
        template <typename T>
        __device__ inline Raw8<T> load8(T const* p)
        {
            Raw8<T> r;
#pragma unroll
            for(int i = 0; i < int(sizeof(T) * 8 / 16); ++i)
                reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<uint4 const*>(p)[i];
            return r;
        }

        // Largest |v| of values as the bits of a float: ordered like the values, a NaN above the
        // infinity.  16-bit types compare two magnitudes at a time, as integers.
        template <typename T>
        __device__ inline uint32_t wordTop(uint32_t top, T const (&v)[2])
        {
            uint32_t w;
            memcpy(&w, v, 4);
            return __vmaxu2(top, w & 0x7fff7fffu);
        }
        __device__ inline float topFloat(uint32_t bits, __half)
        {
            return __half2float(__ushort_as_half(uint16_t(bits)));
        }
        __device__ inline float topFloat(uint32_t bits, __nv_bfloat16)
        {
            return __uint_as_float(bits << 16);
        }
        // A running maximum; merged over lanes or places, then turned into a float.
        template <typename T>
        struct Top
        {
            uint32_t bits = 0;
            __device__ void two(T a, T b)
            {
                if constexpr(sizeof(T) == 2)
                {
                    const T v[2] = {a, b};
                    bits         = wordTop(bits, v);
                }
                else
                    bits = max(bits, max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
            }
            __device__ void lanes(uint32_t with)
            {
                const uint32_t other = __shfl_xor_sync(0xffffffffu, bits, with);
                if constexpr(sizeof(T) == 2)
                    bits = __vmaxu2(bits, other);
                else
                    bits = max(bits, other);
            }
            __device__ float value() const
            {
                if constexpr(sizeof(T) == 2)
                    return topFloat(max(bits & 0xffffu, bits >> 16), T());
                else
                    return __uint_as_float(bits);
            }
        };

        // The scale of a block whose largest magnitude is `top`.
        struct Scale
        {
            uint32_t byte;
            float    inverse; // MXF4: exactly 1 / s; NVF4: 1 / s rounded; 0: codes are zero
            float    value;
        };
        template <bool NV>
        __device__ inline Scale scaleOf(float top)
        {
            const bool fine = top < __uint_as_float(0x7f800000u); // false for a NaN
            Scale      s;
            if constexpr(NV)
            {
                const uint32_t byte = toE4m3(fminf(__fdiv_rn(fine ? top : 0.0f, 6.0f), 448.0f));
                s.value             = fromE4m3(byte);
                s.inverse           = byte != 0u ? __frcp_rn(s.value) : 0.0f;
                s.byte              = fine ? byte : 0x7fu;
            }
            else
            {
                const uint32_t e    = __float_as_uint(fine ? top : 0.0f) >> 23;
                const uint32_t byte = e > 2u ? e - 2u : 0u;
                s.value             = 0.0f;
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

        // Eight codes.  (A NaN or an infinity times an inverse of zero would not give codes of zero:
        // those of such blocks are cleared as words.)
        template <typename T, bool NV>
        __device__ inline uint32_t codes8(T const (&x)[8], Scale const& s, float factor)
        {
            float v[8];
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[i] = toFloat(x[i]);
            if(factor != 1.0f)
            {
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    v[i] *= factor;
            }
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[i] = scaledBy<T, NV>(v[i], s);
            const uint32_t c = e2m1x8(v);
            return s.inverse != 0.0f ? c : 0u;
        }

        // Byte of (row, block) in a scale tile of its row.
        __device__ inline uint32_t scaleOffset(uint32_t row, uint32_t block)
        {
            return (block / 4u) * MX_TILE_BYTES + (row % 32u) * 16u + (row / 32u % 4u) * 4u
                   + block % 4u;
        }

        // A row of a tile whose values do not start on 16-byte boundaries in global memory passes
        // through shared memory, where it lies as far from a boundary as it does there: whole
        // 16-byte pieces move as such, only those that the row shares with its neighbours or with
        // the next tile move value by value.
        template <typename T>
        struct StagedRow
        {
            static constexpr uint32_t PER   = 16 / sizeof(T); // values of a piece
            static constexpr uint32_t PITCH = (TILE_K + PER) * sizeof(T);
            static constexpr uint32_t PIECES = TILE_K / PER + 1u;

            static __device__ uint32_t shift(T const* row)
            {
                return uint32_t(reinterpret_cast<uintptr_t>(row) % 16u) / uint32_t(sizeof(T));
            }
        };
        // Threads of the block move rows of `count` values, row r of the tile at global(r), to or
        // from shared memory.
        template <typename T, bool LOAD, typename Row>
        __device__ inline void moveStaged(uint8_t* staged, uint32_t rows, uint32_t count, Row global)
        {
            using S = StagedRow<T>;
            for(uint32_t i = threadIdx.x; i < rows * S::PIECES; i += THREADS)
            {
                const uint32_t r = i / S::PIECES, piece = i % S::PIECES;
                T*             row   = global(r);
                const uint32_t shift = S::shift(row);
                const uint32_t first = piece * S::PER; // of the piece, counted from the boundary
                T*             here  = reinterpret_cast<T*>(staged + r * S::PITCH) + first;
                T*             there = row + (int32_t(first) - int32_t(shift));
                if(first >= shift && first + S::PER <= shift + count)
                {
                    if(LOAD)
                        *reinterpret_cast<uint4*>(here) = *reinterpret_cast<uint4 const*>(there);
                    else
                        *reinterpret_cast<uint4*>(there) = *reinterpret_cast<uint4 const*>(here);
                }
                else
                {
#pragma unroll
                    for(uint32_t j = 0; j < S::PER; ++j)
                        if(first + j >= shift && first + j < shift + count)
                        {
                            if(LOAD)
                                here[j] = there[j];
                            else
                                there[j] = here[j];
                        }
                }
            }
        }

        struct QuantizeParams
        {
            void const* x;
            uint8_t*    codes;
            uint8_t*    scales;
            uint64_t    ldq; // bytes
            uint64_t    ldx; // elements
            uint32_t    rows, k, groups, tilesK;
            uint32_t    tilesPerBlock; // rows only
            float       factor; // 2^-exponent
        };

        // Columns that a block's threads take at a time, and how many such tiles a block has: more of
        // them spread what a block sets up over more values, but the device is filled first.
        inline uint32_t tilesPerBlock(uint64_t tiles, uint32_t tilesK)
        {
            const uint64_t per = tiles / (2u * 8u * 148u); // eight blocks to an SM, twice
            return uint32_t(per < 1u ? 1u : per > 8u ? 8u : per < tilesK ? per : tilesK);
        }

        // x row-major: k is contiguous.  A block takes 32 rows x 128 columns at a time: sixteen
        // threads read 128 values of a row, eight each, and a block's largest magnitude comes from
        // its two (NVF4) or four (MXF4) threads; those with the scales of four blocks write them as
        // a word.  The values of the next tile are on their way while those of one are worked on.
        template <typename T, bool NV, bool VEC>
        __global__ void __launch_bounds__(THREADS) quantizeRowsKernel(const QuantizeParams p)
        {
            constexpr uint32_t STEPS  = SLAB_ROWS / (THREADS / 16);
            constexpr uint32_t GROUPS = TILE_K / (4u * mxBlock(NV)), LANES = mxBlock(NV) / 8u; // of a block
            const uint32_t across = (p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock;
            const uint32_t slab = blockIdx.x / across, tile0 = blockIdx.x % across * p.tilesPerBlock;
            const uint32_t tiles = min(p.tilesPerBlock, p.tilesK - tile0);
            const uint32_t col = threadIdx.x % 16u * 8u, rowIn = threadIdx.x / 16u;
            const uint64_t row0 = uint64_t(slab) * SLAB_ROWS;
            const uint32_t rows = row0 < p.rows ? uint32_t(min(uint64_t(SLAB_ROWS), p.rows - row0)) : 0u;
            // this thread's places in its rows: rowIn and rowIn + 16
            T const*       x[STEPS];
            uint8_t*       codes[STEPS];
            uint8_t*       scales[STEPS];
            const uint64_t k0 = uint64_t(tile0) * TILE_K + col;
#pragma unroll
            for(uint32_t i = 0; i < STEPS; ++i)
            {
                const uint32_t r = i * 16u + rowIn;
                x[i]      = static_cast<T const*>(p.x) + (row0 + r) * p.ldx + k0;
                codes[i]  = p.codes + (row0 + r) * p.ldq + k0 / 2u;
                scales[i] = p.scales + (uint64_t(slab / 4u) * p.groups + k0 / (4u * mxBlock(NV))) * MX_TILE_BYTES
                            + scaleOffset(slab % 4u * SLAB_ROWS + r, 0);
            }
            uint32_t       left  = p.k > k0 ? uint32_t(p.k - k0) : 0u; // columns from the thread's first on
            uint32_t       pitch = mxPitch(p.k) > k0 / 2u ? uint32_t(mxPitch(p.k) - k0 / 2u) : 0u; // bytes
            uint32_t       group = uint32_t(k0 / (4u * mxBlock(NV)));
            __shared__ alignas(16) uint8_t staged[VEC ? 16 : SLAB_ROWS * StagedRow<T>::PITCH];
            auto fetch = [&](uint32_t t, Raw8<T>(&raw)[STEPS]) {
                const uint32_t done = t * TILE_K;
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                    raw[i] = zero8<T>();
                if constexpr(VEC)
                {
#pragma unroll
                    for(uint32_t i = 0; i < STEPS; ++i)
                        if(i * 16u + rowIn < rows && left >= done + 8u)
                            raw[i] = load8(x[i] + done);
                    if(left > done && left < done + 8u)
                    {
#pragma unroll
                        for(uint32_t i = 0; i < STEPS; ++i)
#pragma unroll
                            for(uint32_t j = 0; j < 8u; ++j)
                                if(i * 16u + rowIn < rows && done + j < left)
                                    raw[i].v[j] = x[i][done + j];
                    }
                }
                else
                {
                    const uint32_t count = min(TILE_K, p.k - (tile0 + t) * TILE_K);
                    auto rowAt = [&](uint32_t r) {
                        return const_cast<T*>(static_cast<T const*>(p.x)) + (row0 + r) * p.ldx + uint64_t(tile0 + t) * TILE_K;
                    };
                    __syncthreads();
                    moveStaged<T, true>(staged, rows, count, rowAt);
                    __syncthreads();
#pragma unroll
                    for(uint32_t i = 0; i < STEPS; ++i)
                    {
                        const uint32_t r = i * 16u + rowIn;
                        if(r < rows)
                        {
                            T const* at = reinterpret_cast<T const*>(staged + r * StagedRow<T>::PITCH)
                                          + StagedRow<T>::shift(rowAt(r)) + col;
#pragma unroll
                            for(uint32_t j = 0; j < 8u; ++j)
                                if(col + j < count)
                                    raw[i].v[j] = at[j];
                        }
                    }
                }
            };
            grid_dependency_wait();
            grid_launch_dependents();
            Raw8<T> raw[STEPS], next[STEPS];
            fetch(0, next);
            for(uint32_t t = 0; t < tiles; ++t)
            {
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                    raw[i] = next[i];
                if(t + 1u < tiles)
                    fetch(t + 1u, next);
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                {
                    Top<T> top;
#pragma unroll
                    for(int j = 0; j < 8; j += 2)
                        top.two(raw[i].v[j], raw[i].v[j + 1]);
                    top.lanes(1);
                    if constexpr(!NV)
                        top.lanes(2);
                    const Scale    s    = scaleOf<NV>(top.value() * p.factor);
                    const uint32_t code = codes8<T, NV>(raw[i].v, s, p.factor);
                    if(i * 16u + rowIn < rows && t * (TILE_K / 2u) < pitch)
                        *reinterpret_cast<uint32_t*>(codes[i] + t * (TILE_K / 2u)) = code;
                    // the bytes of four blocks, a word of the scale tile's row
                    uint32_t word = s.byte << (8u * (threadIdx.x / LANES % 4u));
                    word |= __shfl_xor_sync(0xffffffffu, word, LANES);
                    word |= __shfl_xor_sync(0xffffffffu, word, 2u * LANES);
                    if(threadIdx.x % (4u * LANES) == 0u && group + t * GROUPS < p.groups)
                        *reinterpret_cast<uint32_t*>(scales[i] + t * (GROUPS * MX_TILE_BYTES)) = word;
                }
            }
        }

        // x column-major: the rows are contiguous.  A block takes 128 rows x four blocks of k (a scale
        // tile), a thread two neighbouring rows and one block of k of each, so that a warp reads 64
        // consecutive values at a time and no maximum crosses a thread; the codes pass through
        // shared memory to leave as rows, the scale tile to leave whole.
        template <typename T, bool NV, bool VEC>
        __global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 4 : 3) quantizeColumnsKernel(const QuantizeParams p)
        {
            constexpr uint32_t B     = mxBlock(NV);
            constexpr uint32_t BYTES = 4 * B / 2, PITCH = BYTES + 16; // of a staged row of codes
            __shared__ alignas(16) uint8_t scales[MX_TILE_BYTES];
            __shared__ alignas(16) uint8_t staged[128 * PITCH];
            struct alignas(2 * sizeof(T)) Pair
            {
                T v[2];
            };
            const uint32_t tileRow = blockIdx.x / p.groups, group = blockIdx.x % p.groups;
            const uint32_t r = threadIdx.x % 64u * 2u, blockIn = threadIdx.x / 64u;
            const uint64_t row = uint64_t(tileRow) * 128u + r, k0 = (uint64_t(group) * 4u + blockIn) * B;
            const uint32_t count = k0 < p.k ? uint32_t(min(uint64_t(B), p.k - k0)) : 0u;
            grid_dependency_wait();
            grid_launch_dependents();
            Pair     v[B];
            T const* x = static_cast<T const*>(p.x) + row + k0 * p.ldx;
#pragma unroll
            for(uint32_t i = 0; i < B; ++i)
                v[i].v[0] = v[i].v[1] = T(0.0f);
            if(VEC && row + 1u < p.rows)
            {
#pragma unroll
                for(uint32_t i = 0; i < B; ++i)
                    if(i < count)
                        v[i] = *reinterpret_cast<Pair const*>(x + i * p.ldx);
            }
            else
            {
                const bool one = row < p.rows, two = row + 1u < p.rows;
#pragma unroll
                for(uint32_t i = 0; i < B; ++i)
                {
                    if(i < count && one)
                        v[i].v[0] = x[i * p.ldx];
                    if(i < count && two)
                        v[i].v[1] = x[i * p.ldx + 1u];
                }
            }
#pragma unroll
            for(int j = 0; j < 2; ++j)
            {
                Top<T> top;
#pragma unroll
                for(uint32_t i = 0; i < B; i += 2)
                    top.two(v[i].v[j], v[i + 1].v[j]);
                const Scale s = scaleOf<NV>(top.value() * p.factor);
                uint32_t    words[B / 8];
#pragma unroll
                for(uint32_t w = 0; w < B / 8; ++w)
                {
                    T y[8];
#pragma unroll
                    for(uint32_t i = 0; i < 8; ++i)
                        y[i] = v[w * 8 + i].v[j];
                    words[w] = codes8<T, NV>(y, s, p.factor);
                }
                scales[scaleOffset(r + j, blockIn)] = uint8_t(s.byte);
                uint32_t* to = reinterpret_cast<uint32_t*>(staged + (r + j) * PITCH + blockIn * (B / 2));
#pragma unroll
                for(uint32_t w = 0; w < B / 8; ++w)
                    to[w] = words[w];
            }
            __syncthreads();
            const uint32_t at = threadIdx.x * 16u;
            if(at < MX_TILE_BYTES)
                *reinterpret_cast<uint4*>(p.scales + (uint64_t(tileRow) * p.groups + group) * MX_TILE_BYTES + at)
                    = *reinterpret_cast<uint4 const*>(scales + at);
            // sixteen bytes a thread
            constexpr uint32_t PIECES = BYTES / 16u;
            const uint64_t     pitch  = mxPitch(p.k);
#pragma unroll
            for(uint32_t i = threadIdx.x; i < 128u * PIECES; i += THREADS)
            {
                const uint32_t rr  = i / PIECES;
                const uint64_t col = uint64_t(group) * BYTES + i % PIECES * 16u, out = uint64_t(tileRow) * 128u + rr;
                if(out < p.rows && col < pitch)
                    *reinterpret_cast<uint4*>(p.codes + out * p.ldq + col)
                        = *reinterpret_cast<uint4 const*>(staged + rr * PITCH + i % PIECES * 16u);
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
            uint32_t       tilesPerBlock;
            float          factor; // 2^exponent
        };

        // Eight values: code * s is exact (three bits times at most four); so is the power of two, short
        // of the subnormals.
        template <typename T, bool NV>
        __device__ inline Raw8<T> values8(uint32_t codes, uint32_t byte, float factor)
        {
            const float s = NV ? fromE4m3(byte) : fromE8m0(byte);
            float       v[8];
            e2m1x8ToFloat(codes, v);
#pragma unroll
            for(int j = 0; j < 8; ++j)
                v[j] *= s;
            if(factor != 1.0f)
            {
#pragma unroll
                for(int j = 0; j < 8; ++j)
                    v[j] *= factor;
            }
            Raw8<T> o;
            if constexpr(std::is_same<T, float>::value)
            {
#pragma unroll
                for(int j = 0; j < 8; ++j)
                    o.v[j] = v[j];
            }
            else
            {
#pragma unroll
                for(int j = 0; j < 8; j += 2)
                    if constexpr(std::is_same<T, __half>::value)
                        reinterpret_cast<__half2*>(&o)[j / 2] = __floats2half2_rn(v[j], v[j + 1]);
                    else
                        reinterpret_cast<__nv_bfloat162*>(&o)[j / 2] = __floats2bfloat162_rn(v[j], v[j + 1]);
            }
            return o;
        }

        // A block takes 32 rows x 128 columns at a time, a thread eight codes of two rows; the codes
        // of the next tile are on their way meanwhile.
        template <typename T, bool NV, bool VEC>
        __global__ void __launch_bounds__(THREADS) dequantizeKernel(const DequantizeParams p)
        {
            constexpr uint32_t STEPS  = SLAB_ROWS / (THREADS / 16);
            constexpr uint32_t GROUPS = TILE_K / (4u * mxBlock(NV));
            const uint32_t across = (p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock;
            const uint32_t slab = blockIdx.x / across, tile0 = blockIdx.x % across * p.tilesPerBlock;
            const uint32_t tiles = min(p.tilesPerBlock, p.tilesK - tile0);
            const uint32_t col = threadIdx.x % 16u * 8u, rowIn = threadIdx.x / 16u;
            const uint64_t row0 = uint64_t(slab) * SLAB_ROWS, k0 = uint64_t(tile0) * TILE_K + col;
            const uint32_t rows = row0 < p.rows ? uint32_t(min(uint64_t(SLAB_ROWS), p.rows - row0)) : 0u;
            const uint32_t left = p.k > k0 ? uint32_t(p.k - k0) : 0u; // columns from the thread's first on
            uint8_t const* codes[STEPS];
            uint8_t const* scales[STEPS];
            T*             out[STEPS];
#pragma unroll
            for(uint32_t i = 0; i < STEPS; ++i)
            {
                const uint32_t r = i * 16u + rowIn;
                codes[i]  = p.codes + (row0 + r) * p.ldq + k0 / 2u;
                scales[i] = p.scales + (uint64_t(slab / 4u) * p.groups + k0 / (4u * mxBlock(NV))) * MX_TILE_BYTES
                            + scaleOffset(slab % 4u * SLAB_ROWS + r, uint32_t(k0 / mxBlock(NV) % 4u));
                out[i] = static_cast<T*>(p.out) + (row0 + r) * p.ldo + k0;
            }
            auto fetch = [&](uint32_t t, uint32_t(&word)[STEPS], uint32_t(&byte)[STEPS]) {
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                {
                    word[i] = byte[i] = 0;
                    if(i * 16u + rowIn < rows && left > t * TILE_K)
                    {
                        word[i] = *reinterpret_cast<uint32_t const*>(codes[i] + t * (TILE_K / 2u));
                        byte[i] = scales[i][t * (GROUPS * MX_TILE_BYTES)];
                    }
                }
            };
            __shared__ alignas(16) uint8_t staged[VEC ? 16 : SLAB_ROWS * StagedRow<T>::PITCH];
            grid_dependency_wait();
            grid_launch_dependents();
            uint32_t word[STEPS], byte[STEPS], nextWord[STEPS], nextByte[STEPS];
            fetch(0, nextWord, nextByte);
            for(uint32_t t = 0; t < tiles; ++t)
            {
                const uint32_t done = t * TILE_K;
#pragma unroll
                for(uint32_t i = 0; i < STEPS; ++i)
                {
                    word[i] = nextWord[i];
                    byte[i] = nextByte[i];
                }
                if(t + 1u < tiles)
                    fetch(t + 1u, nextWord, nextByte);
                if constexpr(VEC)
                {
#pragma unroll
                    for(uint32_t i = 0; i < STEPS; ++i)
                    {
                        const Raw8<T> o  = values8<T, NV>(word[i], byte[i], p.factor);
                        T*            at = out[i] + done;
                        if(i * 16u + rowIn >= rows || left <= done)
                            continue;
                        if(left >= done + 8u)
                        {
#pragma unroll
                            for(int j = 0; j < int(sizeof(T) * 8 / 16); ++j)
                                reinterpret_cast<uint4*>(at)[j] = reinterpret_cast<uint4 const*>(&o)[j];
                        }
                        else
                        {
#pragma unroll
                            for(uint32_t j = 0; j < 8u; ++j)
                                if(done + j < left)
                                    at[j] = o.v[j];
                        }
                    }
                }
                else
                {
                    const uint32_t count = min(TILE_K, p.k - (tile0 + t) * TILE_K);
                    auto rowAt = [&](uint32_t r) {
                        return static_cast<T*>(p.out) + (row0 + r) * p.ldo + uint64_t(tile0 + t) * TILE_K;
                    };
                    __syncthreads();
#pragma unroll
                    for(uint32_t i = 0; i < STEPS; ++i)
                    {
                        const uint32_t r = i * 16u + rowIn;
                        const Raw8<T>  o = values8<T, NV>(word[i], byte[i], p.factor);
                        if(r < rows)
                        {
                            T* at = reinterpret_cast<T*>(staged + r * StagedRow<T>::PITCH) + StagedRow<T>::shift(rowAt(r)) + col;
#pragma unroll
                            for(int j = 0; j < 8; ++j)
                                at[j] = o.v[j];
                        }
                    }
                    __syncthreads();
                    moveStaged<T, false>(staged, rows, count, rowAt);
                }
            }
        }

        bool aligned(void const* p, uint64_t bytes)
        {
            return reinterpret_cast<uintptr_t>(p) % bytes == 0;
        }

        // Slabs of 32 rows that hold a row, or (`whole`) whose scales are written: those of whole
        // tiles of 128.
        uint32_t slabsOf(uint32_t rows, bool whole)
        {
            return whole ? mxRowTiles(rows) * 4u : uint32_t((uint64_t(rows) + SLAB_ROWS - 1u) / SLAB_ROWS);
        }

        template <typename T>
        int quantize(bool nv, bool columns, QuantizeParams p, cudaStream_t stream)
        {
            // Wide loads where every row (or pair of rows) starts on their boundary.
            const uint64_t width = columns ? 2 * sizeof(T) : 16;
            const bool     vec   = aligned(p.x, width) && p.ldx * sizeof(T) % width == 0;
            const uint32_t slabs = slabsOf(p.rows, true);
            p.tilesPerBlock      = tilesPerBlock(uint64_t(slabs) * p.tilesK, p.tilesK);
            const uint32_t blocks = columns ? mxRowTiles(p.rows) * p.groups
                                            : slabs * ((p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock);
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
        int dequantize(bool nv, DequantizeParams p, cudaStream_t stream)
        {
            const bool     vec   = aligned(p.out, 16) && p.ldo * sizeof(T) % 16 == 0;
            const uint32_t slabs = slabsOf(p.rows, false);
            p.tilesPerBlock      = tilesPerBlock(uint64_t(slabs) * p.tilesK, p.tilesK);
            const uint32_t blocks = slabs * ((p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock);
            auto launch = [&](auto kernel) {
                return cudaToStatus(launchOverlapped(kernel, dim3(blocks), dim3(THREADS), 0, stream, p));
            };
            return nv ? (vec ? launch(dequantizeKernel<T, true, true>) : launch(dequantizeKernel<T, true, false>))
                      : (vec ? launch(dequantizeKernel<T, false, true>) : launch(dequantizeKernel<T, false, false>));
        }

        // What both directions check; OK or a status.
        int checkOperand(int fmt, int dtype, uint32_t rows, uint32_t k, void const* values,
                         uint64_t ld, uint64_t span, int exponent, void const* codes, uint64_t ldq,
                         void const* scales)
        {
            if(!values || !codes || !scales || rows == 0 || k == 0 || ld < span || ldq < mxPitch(k)
               || exponent < -64 || exponent > 64)
                return B200WMMA_ERR_INVALID_ARG;
            if(!mxFormat(fmt) || (dtype != B200WMMA_F16 && dtype != B200WMMA_BF16 && dtype != B200WMMA_F32))
                return B200WMMA_ERR_UNSUPPORTED;
            if(!aligned(codes, 16) || !aligned(scales, 16) || ldq % 16 || !aligned(values, dtypeSize(dtype)))
                return B200WMMA_ERR_ALIGNMENT;
            // blocks of a launch, four slabs to a tile of 128 rows
            if(uint64_t(mxRowTiles(rows)) * ((uint64_t(k) + TILE_K - 1) / TILE_K) > 0x1fffffffull)
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
    const int rc = checkOperand(fmt, in_dtype, rows, k, x, ldx, columns ? rows : k, exponent, codes,
                                ldq, scales);
    if(rc != B200WMMA_OK)
        return rc;
    const bool           nv = fmt == B200WMMA_NVF4;
    const QuantizeParams p{x, static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), ldq, ldx,
                           rows, k, mxGroups(nv, k), uint32_t((uint64_t(k) + TILE_K - 1) / TILE_K),
                           0, ldexpf(1.0f, -exponent)};
    const cudaStream_t   s = static_cast<cudaStream_t>(stream);
    switch(in_dtype)
    {
    case B200WMMA_F16:
        return quantize<__half>(nv, columns, p, s);
    case B200WMMA_BF16:
        return quantize<__nv_bfloat16>(nv, columns, p, s);
    }
    return quantize<float>(nv, columns, p, s);
}

int b200wmma_mx_dequantize(int fmt, int out_dtype, uint32_t rows, uint32_t k, const void* codes,
                           uint64_t ldq, const void* scales, int exponent, void* out, uint64_t ldo,
                           void* stream)
{
    const int rc = checkOperand(fmt, out_dtype, rows, k, out, ldo, k, exponent, codes, ldq, scales);
    if(rc != B200WMMA_OK)
        return rc;
    const bool             nv = fmt == B200WMMA_NVF4;
    const DequantizeParams p{static_cast<uint8_t const*>(codes), static_cast<uint8_t const*>(scales),
                             out, ldq, ldo, rows, k, mxGroups(nv, k),
                             uint32_t((uint64_t(k) + TILE_K - 1) / TILE_K), 0, ldexpf(1.0f, exponent)};
    const cudaStream_t     s = static_cast<cudaStream_t>(stream);
    switch(out_dtype)
    {
    case B200WMMA_F16:
        return dequantize<__half>(nv, p, s);
    case B200WMMA_BF16:
        return dequantize<__nv_bfloat16>(nv, p, s);
    }
    return dequantize<float>(nv, p, s);
}
}
