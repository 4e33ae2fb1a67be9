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
// for NVF4 see codes8().
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

        // Sixteen consecutive values of a row as they are stored.
        constexpr uint32_t RUN = 16;
        template <typename T>
        struct alignas(32) Run
        {
            T v[RUN];
        };
        template <typename T>
        __device__ inline Run<T> zeroRun()
        {
            Run<T> r;
#pragma unroll
            for(uint32_t i = 0; i < RUN; ++i)
                r.v[i] = T(0.0f);
            return r;
        }
        // ... moved in words of WIDTH bytes, 32 or 16, whichever boundary the rows lie on.
        template <typename T, int WIDTH>
        __device__ inline Run<T> loadRun(T const* p)
        {
            Run<T> r;
            if constexpr(WIDTH == 32)
            {
                uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
                for(uint32_t i = 0; i < sizeof(r) / 4u; i += 8u)
                    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                 : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]),
                                   "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                                 : "l"(reinterpret_cast<uint32_t const*>(p) + i));
            }
            else
            {
#pragma unroll
                for(uint32_t i = 0; i < sizeof(r) / 16u; ++i)
                    reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<uint4 const*>(p)[i];
            }
            return r;
        }
        template <typename T, int WIDTH>
        __device__ inline void storeRun(T* p, Run<T> const& r)
        {
            if constexpr(WIDTH == 32)
            {
                uint32_t const* w = reinterpret_cast<uint32_t const*>(&r);
#pragma unroll
                for(uint32_t i = 0; i < sizeof(r) / 4u; i += 8u)
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(reinterpret_cast<uint32_t*>(p) + i),
                                 "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]),
                                 "r"(w[i + 6]), "r"(w[i + 7])
                                 : "memory");
            }
            else
            {
#pragma unroll
                for(uint32_t i = 0; i < sizeof(r) / 16u; ++i)
                    reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<uint4 const*>(&r)[i];
            }
        }

        // Values are worked on as the 32-bit words they come in, two to a word if they have 16 bits:
        // taken out one by one, they cost twice the instructions that the arithmetic does.
        template <typename T>
        struct Words
        {
            static constexpr uint32_t PER = 4 / sizeof(T); // values of a word
            static __device__ float value(uint32_t w, uint32_t) // of 32 bits
            {
                return __uint_as_float(w);
            }
            // running maximum of magnitudes, place by place; a NaN stays one
            static __device__ uint32_t top(uint32_t most, uint32_t w)
            {
                return max(most, w & 0x7fffffffu);
            }
        };
        template <typename T, typename T2>
        struct Words16
        {
            static constexpr uint32_t PER = 2;
            static __device__ uint32_t top(uint32_t most, uint32_t w)
            {
                const T2 m = __hmax2_nan(*reinterpret_cast<T2*>(&most), __habs2(*reinterpret_cast<T2*>(&w)));
                return *reinterpret_cast<uint32_t const*>(&m);
            }
        };
        template <>
        struct Words<__nv_bfloat16> : Words16<__nv_bfloat16, __nv_bfloat162>
        {
            static __device__ float value(uint32_t w, uint32_t place)
            {
                return __uint_as_float(place ? w & 0xffff0000u : w << 16);
            }
        };
        template <>
        struct Words<__half> : Words16<__half, __half2>
        {
            static __device__ float value(uint32_t w, uint32_t place)
            {
                const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
                return place ? f.y : f.x;
            }
        };

        // The scale of a block whose largest magnitude is `top`, for values x with y = x * factor.
        struct Scale
        {
            uint32_t byte;
            float    times; // factor / s (NVF4: 1 / s rounded); 0: codes are zero
            float    value;
        };
        template <bool NV>
        __device__ inline Scale scaleOf(float top, float factor)
        {
            const float y    = top * factor;
            const bool  fine = y < __uint_as_float(0x7f800000u); // false for a NaN
            Scale       s;
            if constexpr(NV)
            {
                const uint32_t byte = toE4m3(fminf(__fdiv_rn(fine ? y : 0.0f, 6.0f), 448.0f));
                s.value             = fromE4m3(byte);
                s.times             = byte != 0u ? __frcp_rn(s.value) * factor : 0.0f;
                s.byte              = fine ? byte : 0x7fu;
            }
            else
            {
                const uint32_t e    = __float_as_uint(fine ? y : 0.0f) >> 23;
                const uint32_t byte = e > 2u ? e - 2u : 0u;
                s.value             = 0.0f;
                s.times = fine ? __uint_as_float((254u - byte) << 23) * factor : 0.0f;
                s.byte  = fine ? byte : 255u;
            }
            return s;
        }
        // Whether x * times is (x * factor) / s: not where times, about 4 / top, left fp32's range, as it
        // does for blocks of values below 2^-125 with a factor of more than one.
        __device__ inline bool safe(Scale const& s)
        {
            const uint32_t e = __float_as_uint(s.times) >> 23;
            return e - 1u < 254u || s.times == 0.0f;
        }

        // Eight values to codes: y / s, exact as far as the rounding to E2M1 can see.  MXF4 divides by a
        // power of two.  For NVF4 the borders between two codes are multiples m s of a 4-bit s by a
        // 3-bit m: at most seven significant bits.  A quotient from 16-bit values (at most eleven
        // bits) is on a border or at least 2^-11 of its size away from it, so x * (1 / s), which is
        // off by less than 2^-22, is rounded to 14 bits: what lay on a border is there again, and
        // nothing else gets there.  For 32-bit values the division is rounded correctly, which
        // keeps the order to every border.
        // (A NaN or an infinity times zero would not give codes of zero: those of blocks without a
        // usable scale are cleared as words.)
        template <typename T, bool NV>
        __device__ inline uint32_t codes8(float (&v)[8], Scale const& s, float factor)
        {
#pragma unroll
            for(int i = 0; i < 8; ++i)
            {
                if constexpr(!NV)
                    v[i] *= s.times;
                else if constexpr(sizeof(T) == 2)
                    v[i] = __uint_as_float((__float_as_uint(v[i] * s.times) + 0x200u) & ~0x3ffu);
                else
                    v[i] = s.times != 0.0f ? __fdiv_rn(v[i] * factor, s.value) : 0.0f;
            }
            const uint32_t c = e2m1x8(v);
            return s.times != 0.0f ? c : 0u;
        }
        // The same in two steps, for blocks that safe() excludes.
        template <bool NV>
        __device__ inline uint32_t codes8Slow(float (&v)[8], Scale const& s, float factor)
        {
            Scale one = s;
            one.times = NV ? 1.0f : __uint_as_float((254u - s.byte) << 23);
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[i] = NV ? __fdiv_rn(v[i] * factor, s.value) : v[i] * factor;
            return codes8<float, false>(v, one, 1.0f);
        }

        // Eight values as words to codes, for blocks that safe() admits.
        template <typename T, bool NV>
        __device__ inline uint32_t codesOf(uint32_t const* w, Scale const& s, float factor)
        {
            using W = Words<T>;
            float v[8];
            if constexpr(std::is_same<T, __nv_bfloat16>::value && !NV)
            {
                // times a power of two, two at a time: exact in bf16 (short of its subnormals, whose
                // codes are zero)
                const __nv_bfloat162 times = __float2bfloat162_rn(s.times); // exactly
#pragma unroll
                for(uint32_t j = 0; j < 4; ++j)
                {
                    const __nv_bfloat162 y  = __hmul2(*reinterpret_cast<__nv_bfloat162 const*>(&w[j]), times);
                    const uint32_t       yw = *reinterpret_cast<uint32_t const*>(&y);
                    v[2 * j]                = W::value(yw, 0);
                    v[2 * j + 1]            = W::value(yw, 1);
                }
                const uint32_t c = e2m1x8(v);
                return s.times != 0.0f ? c : 0u;
            }
            else
            {
#pragma unroll
                for(uint32_t j = 0; j < 8; ++j)
                    v[j] = W::value(w[j / W::PER], j % W::PER);
                return codes8<T, NV>(v, s, factor);
            }
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
        // The eight threads of a row (`lane` 0 to 7) move `count` values of it to or from shared memory.
        template <typename T, bool LOAD>
        __device__ inline void moveStaged(uint8_t* staged, T* row, uint32_t shift, uint32_t count, uint32_t lane)
        {
            using S = StagedRow<T>;
#pragma unroll
            for(uint32_t i = 0; i < (S::PIECES + 7u) / 8u; ++i)
            {
                const uint32_t first = (i * 8u + lane) * S::PER; // of the piece, counted from the boundary
                T*             here  = reinterpret_cast<T*>(staged) + first;
                T*             there = row + (int32_t(first) - int32_t(shift));
                if(first >= shift && first + S::PER <= shift + count)
                {
                    if(LOAD)
                        *reinterpret_cast<uint4*>(here) = *reinterpret_cast<uint4 const*>(there);
                    else
                        *reinterpret_cast<uint4*>(there) = *reinterpret_cast<uint4 const*>(here);
                }
                else if(first < shift + count)
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

        // x row-major: k is contiguous.  A block takes 32 rows x 128 columns at a time: eight threads
        // have 128 values of a row, sixteen each, which is a block (NVF4) or half of one (MXF4);
        // those with the scales of four blocks write them as a word.  The values of the next tile
        // are on their way while those of one are worked on.  (8192 x 8192 bf16 MXF4, 171 MB: 34 us; 26 at the
        // measured copy rate; 64 with eight values a thread and maxima found as integers.)
        template <typename T, bool NV, int WIDTH>
        __global__ void __launch_bounds__(THREADS) quantizeRowsKernel(const QuantizeParams p)
        {
            using W                   = Words<T>;
            constexpr uint32_t GROUPS = TILE_K / (4u * mxBlock(NV)), LANES = mxBlock(NV) / RUN; // of a block
            const uint32_t across = (p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock;
            const uint32_t slab = blockIdx.x / across, tile0 = blockIdx.x % across * p.tilesPerBlock;
            const uint32_t tiles = min(p.tilesPerBlock, p.tilesK - tile0);
            const uint32_t col = threadIdx.x % 8u * RUN, r = threadIdx.x / 8u;
            const uint64_t row0 = uint64_t(slab) * SLAB_ROWS, row = row0 + r, k0 = uint64_t(tile0) * TILE_K + col;
            const uint32_t rows = row0 < p.rows ? uint32_t(min(uint64_t(SLAB_ROWS), p.rows - row0)) : 0u;
            T const*       x      = static_cast<T const*>(p.x) + row * p.ldx + k0;
            uint8_t*       codes  = p.codes + row * p.ldq + k0 / 2u;
            uint8_t*       scales = p.scales + (uint64_t(slab / 4u) * p.groups + k0 / (4u * mxBlock(NV))) * MX_TILE_BYTES
                              + scaleOffset(slab % 4u * SLAB_ROWS + r, 0);
            const uint32_t left  = r < rows && p.k > k0 ? uint32_t(p.k - k0) : 0u; // values from the first on
            const uint32_t pitch = r < rows && mxPitch(p.k) > k0 / 2u ? uint32_t(mxPitch(p.k) - k0 / 2u) : 0u; // bytes
            const uint32_t group = uint32_t(k0 / (4u * mxBlock(NV)));
            __shared__ alignas(16) uint8_t staged[WIDTH ? 16 : SLAB_ROWS * StagedRow<T>::PITCH];
            auto fetch = [&](uint32_t t) {
                const uint32_t done = t * TILE_K;
                Run<T>         raw;
                if constexpr(WIDTH != 0)
                {
                    if(left >= done + RUN)
                        return loadRun<T, WIDTH>(x + done);
                    raw = zeroRun<T>();
#pragma unroll
                    for(uint32_t j = 0; j < RUN; ++j)
                        if(done + j < left)
                            raw.v[j] = x[done + j];
                }
                else
                {
                    // (a row's threads are in one warp)
                    const uint32_t count = min(TILE_K, p.k - (tile0 + t) * TILE_K);
                    T*             from  = const_cast<T*>(x) - col + done;
                    const uint32_t shift = StagedRow<T>::shift(from);
                    uint8_t*       here  = staged + r * StagedRow<T>::PITCH;
                    __syncwarp();
                    if(r < rows)
                        moveStaged<T, true>(here, from, shift, count, threadIdx.x % 8u);
                    __syncwarp();
                    raw = zeroRun<T>();
                    if(r < rows)
                    {
                        T const* at = reinterpret_cast<T const*>(here) + shift + col;
#pragma unroll
                        for(uint32_t j = 0; j < RUN; ++j)
                            if(col + j < count)
                                raw.v[j] = at[j];
                    }
                }
                return raw;
            };
            grid_dependency_wait();
            grid_launch_dependents();
            Run<T> next = fetch(0);
            for(uint32_t t = 0; t < tiles; ++t)
            {
                const Run<T> raw = next;
                if(t + 1u < tiles)
                    next = fetch(t + 1u);
                uint32_t const* w   = reinterpret_cast<uint32_t const*>(&raw);
                uint32_t        top = 0;
#pragma unroll
                for(uint32_t j = 0; j < RUN / W::PER; ++j)
                    top = W::top(top, w[j]);
                if constexpr(!NV)
                    top = W::top(top, __shfl_xor_sync(0xffffffffu, top, 1));
                if constexpr(W::PER == 2)
                    top = W::top(top, top << 16 | top >> 16);
                const Scale s = scaleOf<NV>(W::value(top, 0), p.factor);
                uint32_t    code[RUN / 8];
                if(safe(s))
                {
#pragma unroll
                    for(uint32_t c = 0; c < RUN / 8; ++c)
                        code[c] = codesOf<T, NV>(w + c * (8 / W::PER), s, p.factor);
                }
                else
                {
#pragma unroll
                    for(uint32_t c = 0; c < RUN / 8; ++c)
                    {
                        float v[8];
#pragma unroll
                        for(uint32_t j = 0; j < 8; ++j)
                            v[j] = W::value(w[(c * 8 + j) / W::PER], j % W::PER);
                        code[c] = codes8Slow<NV>(v, s, p.factor);
                    }
                }
                if(t * (TILE_K / 2u) < pitch)
                    *reinterpret_cast<uint2*>(codes) = make_uint2(code[0], code[1]);
                codes += TILE_K / 2u;
                // the bytes of four blocks, a word of the scale tile's row
                uint32_t word = s.byte << (8u * (threadIdx.x / LANES % 4u));
                word |= __shfl_xor_sync(0xffffffffu, word, LANES);
                word |= __shfl_xor_sync(0xffffffffu, word, 2u * LANES);
                if(threadIdx.x % (4u * LANES) == 0u && group + t * GROUPS < p.groups)
                    *reinterpret_cast<uint32_t*>(scales) = word;
                scales += GROUPS * MX_TILE_BYTES;
            }
        }

        // x column-major: the rows are contiguous.  A block takes 128 rows x four blocks of k (a scale
        // tile), a thread two neighbouring rows and one block of k of each, so that a warp reads 64
        // consecutive values at a time and no maximum crosses a thread; the codes pass through
        // shared memory to leave as rows, the scale tile to leave whole.  (5000 x 4099 f16 NVF4: 15.5 us.)
        template <typename T, bool NV, bool VEC>
        __global__ void __launch_bounds__(THREADS, NV ? 4 : 2) quantizeColumnsKernel(const QuantizeParams p)
        {
            constexpr uint32_t B     = mxBlock(NV);
            constexpr uint32_t BYTES = 4 * B / 2, PITCH = BYTES + 16; // of a staged row of codes
            __shared__ alignas(16) uint8_t scales[MX_TILE_BYTES];
            __shared__ alignas(16) uint8_t staged[128 * PITCH];
            using W = Words<T>;
            constexpr uint32_t PAIR = 2 / W::PER; // words of two values
            struct alignas(2 * sizeof(T)) Pair
            {
                uint32_t w[PAIR];
            };
            static_assert(sizeof(Pair) == 2 * sizeof(T), "two values");
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
                v[i] = Pair{};
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
                    T both[2] = {T(0.0f), T(0.0f)};
                    if(i < count && one)
                        both[0] = x[i * p.ldx];
                    if(i < count && two)
                        both[1] = x[i * p.ldx + 1u];
                    memcpy(&v[i], both, sizeof(both));
                }
            }
            uint32_t tops[PAIR] = {}; // of 16 bits: both rows' in a word
#pragma unroll
            for(uint32_t i = 0; i < B; ++i)
#pragma unroll
                for(uint32_t j = 0; j < PAIR; ++j)
                    tops[j] = W::top(tops[j], v[i].w[j]);
#pragma unroll
            for(uint32_t j = 0; j < 2; ++j)
            {
                const Scale s = scaleOf<NV>(W::value(tops[j / W::PER], j % W::PER), p.factor);
                uint32_t    words[B / 8];
#pragma unroll
                for(uint32_t c = 0; c < B / 8; ++c)
                {
                    float y[8];
#pragma unroll
                    for(uint32_t i = 0; i < 8; ++i)
                        y[i] = W::value(v[c * 8 + i].w[j / W::PER], j % W::PER);
                    words[c] = safe(s) ? codes8<T, NV>(y, s, p.factor) : codes8Slow<NV>(y, s, p.factor);
                }
                scales[scaleOffset(r + j, blockIn)] = uint8_t(s.byte);
                uint32_t* to = reinterpret_cast<uint32_t*>(staged + (r + j) * PITCH + blockIn * (B / 2));
#pragma unroll
                for(uint32_t c = 0; c < B / 8; ++c)
                    to[c] = words[c];
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
            float          factor; // 2^exponent; MXF4: four times that, see scaleValue()
        };

        // A block's scale s; MXF4: s / 4, since 6 * 2^127 is beyond fp32 where 2^exponent can bring it back.
        // (Both s / 4 and half of it are fp32 numbers down to s = 2^-127.)
        template <bool NV>
        __device__ inline float scaleValue(uint32_t byte)
        {
            return NV ? fromE4m3(byte) : 0.25f * fromE8m0(byte);
        }

        // Eight values: code * s is exact (three bits times at most four); so is the power of two, short
        // of the subnormals.
        template <typename T>
        __device__ inline void values8(uint32_t codes, float s, float factor, T* out)
        {
            float v[8];
            e2m1x8ToFloat(codes, v);
#pragma unroll
            for(int j = 0; j < 8; ++j)
                v[j] = v[j] * s * factor;
#pragma unroll
            for(int j = 0; j < 8; j += 2)
                if constexpr(std::is_same<T, __half>::value)
                    reinterpret_cast<__half2*>(out)[j / 2] = __floats2half2_rn(v[j], v[j + 1]);
                else if constexpr(std::is_same<T, __nv_bfloat16>::value)
                    reinterpret_cast<__nv_bfloat162*>(out)[j / 2] = __floats2bfloat162_rn(v[j], v[j + 1]);
                else
                {
                    out[j]     = v[j];
                    out[j + 1] = v[j + 1];
                }
        }

        // A block takes 32 rows x 128 columns at a time, a thread sixteen codes; those of the next
        // tile are on their way meanwhile.  (8192 x 8192 MXF4 to bf16: 31 us, 26 for its bytes.)
        template <typename T, bool NV, int WIDTH>
        __global__ void __launch_bounds__(THREADS) dequantizeKernel(const DequantizeParams p)
        {
            constexpr uint32_t GROUPS = TILE_K / (4u * mxBlock(NV));
            const uint32_t across = (p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock;
            const uint32_t slab = blockIdx.x / across, tile0 = blockIdx.x % across * p.tilesPerBlock;
            const uint32_t tiles = min(p.tilesPerBlock, p.tilesK - tile0);
            const uint32_t col = threadIdx.x % 8u * RUN, r = threadIdx.x / 8u;
            const uint64_t row0 = uint64_t(slab) * SLAB_ROWS, row = row0 + r, k0 = uint64_t(tile0) * TILE_K + col;
            const uint32_t rows = row0 < p.rows ? uint32_t(min(uint64_t(SLAB_ROWS), p.rows - row0)) : 0u;
            const uint32_t left = r < rows && p.k > k0 ? uint32_t(p.k - k0) : 0u; // values from the first on
            uint8_t const* codes  = p.codes + row * p.ldq + k0 / 2u;
            uint8_t const* scales = p.scales + (uint64_t(slab / 4u) * p.groups + k0 / (4u * mxBlock(NV))) * MX_TILE_BYTES
                                    + scaleOffset(slab % 4u * SLAB_ROWS + r, uint32_t(k0 / mxBlock(NV) % 4u));
            T*             out    = static_cast<T*>(p.out) + row * p.ldo + k0;
            __shared__ alignas(16) uint8_t staged[WIDTH ? 16 : SLAB_ROWS * StagedRow<T>::PITCH];
            grid_dependency_wait();
            grid_launch_dependents();
            uint2    nextCode{};
            uint32_t nextByte = 0;
            auto     fetch    = [&](uint32_t t) {
                if(left > t * TILE_K)
                {
                    nextCode = *reinterpret_cast<uint2 const*>(codes + t * (TILE_K / 2u));
                    nextByte = scales[t * (GROUPS * MX_TILE_BYTES)];
                }
            };
            fetch(0);
            for(uint32_t t = 0; t < tiles; ++t)
            {
                const uint32_t done = t * TILE_K;
                const uint2    code = nextCode;
                const float    s    = scaleValue<NV>(nextByte);
                if(t + 1u < tiles)
                    fetch(t + 1u);
                Run<T> o;
                values8<T>(code.x, s, p.factor, o.v);
                values8<T>(code.y, s, p.factor, o.v + 8);
                if constexpr(WIDTH != 0)
                {
                    if(left >= done + RUN)
                        storeRun<T, WIDTH>(out + done, o);
                    else
                    {
#pragma unroll
                        for(uint32_t j = 0; j < RUN; ++j)
                            if(done + j < left)
                                out[done + j] = o.v[j];
                    }
                }
                else
                {
                    const uint32_t count = min(TILE_K, p.k - (tile0 + t) * TILE_K);
                    T*             to    = out - col + done;
                    const uint32_t shift = StagedRow<T>::shift(to);
                    uint8_t*       here  = staged + r * StagedRow<T>::PITCH;
                    __syncwarp();
                    if(r < rows)
                    {
                        T* at = reinterpret_cast<T*>(here) + shift + col;
#pragma unroll
                        for(uint32_t j = 0; j < RUN; ++j)
                            at[j] = o.v[j];
                    }
                    __syncwarp();
                    if(r < rows)
                        moveStaged<T, false>(here, to, shift, count, threadIdx.x % 8u);
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

        // f(32), f(16) or f(0): the boundary that rows `pitch` bytes apart start on; none: through shared
        // memory.  (Rows on 16 bytes, quantised, through shared memory and so: 5335 x 3604 f32 NVF4 51.5 and
        // 24.1 us, 8192 x 8200 bf16 MXF4 65.9 and 37.6.)
        template <typename F>
        int withWidth(void const* base, uint64_t pitch, F f)
        {
            if(aligned(base, 32) && pitch % 32 == 0)
                return f(std::integral_constant<int, 32>());
            if(aligned(base, 16) && pitch % 16 == 0)
                return f(std::integral_constant<int, 16>());
            return f(std::integral_constant<int, 0>());
        }

        template <typename T>
        int quantize(bool nv, bool columns, QuantizeParams p, cudaStream_t stream)
        {
            const uint32_t slabs = slabsOf(p.rows, true);
            p.tilesPerBlock      = tilesPerBlock(uint64_t(slabs) * p.tilesK, p.tilesK);
            const uint32_t blocks = columns ? mxRowTiles(p.rows) * p.groups
                                            : slabs * ((p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock);
            auto launch = [&](auto kernel) {
                return cudaToStatus(launchOverlapped(kernel, dim3(blocks), dim3(THREADS), 0, stream, p));
            };
            if(columns)
            {
                const bool vec = aligned(p.x, 2 * sizeof(T)) && p.ldx % 2 == 0; // pairs of rows
                return nv ? (vec ? launch(quantizeColumnsKernel<T, true, true>) : launch(quantizeColumnsKernel<T, true, false>))
                          : (vec ? launch(quantizeColumnsKernel<T, false, true>) : launch(quantizeColumnsKernel<T, false, false>));
            }
            return withWidth(p.x, p.ldx * sizeof(T), [&](auto width) {
                return nv ? launch(quantizeRowsKernel<T, true, width.value>) : launch(quantizeRowsKernel<T, false, width.value>);
            });
        }

        template <typename T>
        int dequantize(bool nv, DequantizeParams p, cudaStream_t stream)
        {
            const uint32_t slabs = slabsOf(p.rows, false);
            p.tilesPerBlock      = tilesPerBlock(uint64_t(slabs) * p.tilesK, p.tilesK);
            const uint32_t blocks = slabs * ((p.tilesK + p.tilesPerBlock - 1u) / p.tilesPerBlock);
            auto launch = [&](auto kernel) {
                return cudaToStatus(launchOverlapped(kernel, dim3(blocks), dim3(THREADS), 0, stream, p));
            };
            return withWidth(p.out, p.ldo * sizeof(T), [&](auto width) {
                // (sixteen values of 32 bits are four pieces of 16 bytes a thread, 64 bytes apart in each store: half
                // sectors.  5335 x 3604 f32: 24 us so, 19 through shared memory; 8192 x 8200 bf16: 41 and 48.)
                if constexpr(width.value == 16 && sizeof(T) == 4)
                    return nv ? launch(dequantizeKernel<T, true, 0>) : launch(dequantizeKernel<T, false, 0>);
                else
                    return nv ? launch(dequantizeKernel<T, true, width.value>) : launch(dequantizeKernel<T, false, width.value>);
            });
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
                             uint32_t((uint64_t(k) + TILE_K - 1) / TILE_K), 0,
                             ldexpf(1.0f, nv ? exponent : exponent + 2)};
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
