// Embedding lookup and the gradient of its table.
//
//   out[o, i, :] = scale * table[row(o, i), :]
//   grad_table[r, :] = scale * sum of grad[o, i, :] over the tokens (o, i) with row(o, i) = r
//
// Tokens are outer x inner; row(o, i) = first[i] + ids[o, i] where the table is several tables
// one behind the other (first has inner + 1 entries; DLRM's categorical features), ids[o, i]
// otherwise.  An id outside its table (-1 marks padding) reads as a row of zeros and has no
// gradient.
//
// Both are bound by HBM.  The gradient is made without atomics on its values, so that a call's
// result depends on its arguments alone: tokens are sorted by row (a stable radix sort), the
// sorted tokens are cut into chunks, and every run of equal rows in a chunk is summed in token
// order, in fp32.  A run inside one chunk is written at once; the pieces of one that crosses
// chunks are added up by the block that has them, and where it crosses blocks too, each block
// leaves a piece in the workspace and a last kernel joins those.  Rows without a token are cleared by
// blocks of their own beside the others.
#include "common.cuh"
#include "mx_format.cuh"
#include "rocwmma/rocwmma_block.hpp"
#include "row_overlap.h"
#include <cstring>
#include <type_traits>

namespace b200wmma
{
    using rocwmma::block::grid_dependency_wait;
    using rocwmma::block::grid_launch_dependents;

    namespace
    {
        constexpr uint32_t THREADS = 256;
        constexpr uint32_t DEVICE_THREADS = 148u * 2048u; // resident at once
        constexpr uint32_t NO_ROW  = 0x7fffffffu; // no token, or no row of the table
        constexpr uint32_t PASSES  = 0x80000000u; // with a row: a run that fills a chunk and goes on

        // n / d for n < 2^31 by a multiplication: m = ceil(2^(31 + s) / d) with 2^s >= d is off by less
        // than d / 2^(31 + s) of a quotient, too little to reach the next one.
        struct Divisor
        {
            uint32_t d = 1, m = 0, s = 0;
            Divisor() = default;
            explicit Divisor(uint32_t by) : d(by)
            {
                while((1ull << s) < by)
                    ++s;
                m = uint32_t(((1ull << (31u + s)) + by - 1u) / by);
            }
            __device__ uint32_t of(uint32_t n) const // d > 1
            {
                return __umulhi(n, m) >> (s - 1u);
            }
        };

        // The tokens of a call.
        struct Tokens
        {
            void const*    ids;
            int64_t const* first;
            uint64_t       idsOuter, idsInner; // strides, elements
            uint32_t       count, rows;
            Divisor        inner;
            uint32_t       wide; // 64-bit ids
        };

        __device__ inline int64_t idOf(Tokens const& t, uint32_t token, uint32_t& outer, uint32_t& inner)
        {
            outer = token;
            inner = 0;
            if(t.inner.d > 1u)
            {
                outer = t.inner.of(token);
                inner = token - outer * t.inner.d;
            }
            const uint64_t at = uint64_t(outer) * t.idsOuter + uint64_t(inner) * t.idsInner;
            return t.wide ? static_cast<int64_t const*>(t.ids)[at] : int64_t(static_cast<int32_t const*>(t.ids)[at]);
        }
        __device__ inline uint32_t rowOf(Tokens const& t, int64_t id, uint32_t inner)
        {
            int64_t begin = 0, end = t.rows;
            if(t.first)
            {
                begin = t.first[inner];
                end   = t.first[inner + 1];
                if(begin < 0 || end < begin || end > int64_t(t.rows)) // (end - begin must not wrap)
                    return NO_ROW;
            }
            return id >= 0 && id < end - begin ? uint32_t(begin + id) : NO_ROW;
        }
        __device__ inline uint32_t rowOf(Tokens const& t, uint32_t token, uint32_t& outer, uint32_t& inner)
        {
            const int64_t id = idOf(t, token, outer, inner);
            return rowOf(t, id, inner);
        }

        // V neighbouring values of a row, at most 32 bytes, moved as one.
        template <typename T, int V>
        struct alignas(sizeof(T) * V) Piece
        {
            T v[V];
        };
        template <typename T, int V>
        __device__ inline Piece<T, V> loadPiece(T const* at)
        {
            Piece<T, V> p;
            if constexpr(sizeof(p) == 32)
            {
                uint32_t* w = reinterpret_cast<uint32_t*>(&p);
                asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                             : "l"(at));
            }
            else
                p = *reinterpret_cast<Piece<T, V> const*>(at);
            return p;
        }
        template <typename T, int V>
        __device__ inline void storePiece(T* at, Piece<T, V> const& p)
        {
            if constexpr(sizeof(p) == 32)
            {
                uint32_t const* w = reinterpret_cast<uint32_t const*>(&p);
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[0]), "r"(w[1]),
                             "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                             : "memory");
            }
            else
                *reinterpret_cast<Piece<T, V>*>(at) = p;
        }

        // ---- lookup ----------------------------------------------------------------------
        struct LookupParams
        {
            Tokens      t;
            void const* table;
            void*       out;
            uint64_t    ldt, outOuter, outInner;
            uint32_t    pieces, lanesLog2; // pieces of a row; threads side by side on a row
            uint32_t    perBlock; // tokens
            uint32_t    slices; // blocks to a row; 0: rows to a block
            float       scale;
        };

        // Pieces that a thread has in flight.
        constexpr uint32_t lookupUnroll(int V)
        {
            return V == 8 ? 4u : 8u;
        }

        // A block finds the rows of its tokens first, one thread a token, then moves them, U pieces
        // in flight a thread: the same piece of U rows, or, where a block has fewer rows than that
        // (p.slices != 0), U pieces of one row, of which a block has a slice.  (4000 rows of 4954 bf16,
        // out of L2: 84 us the first way, 17 the second; one row of 16384 f16: 4.5 and 1.7.)
        // Bound by HBM: 65536 x 26 x 128 f16 take 83 us, 5.3 TB/s of the 436 MB that are written.
        template <typename T, typename OutT, int V>
        __global__ void __launch_bounds__(THREADS) lookupKernel(const LookupParams p)
        {
            constexpr uint32_t U = lookupUnroll(V);
            __shared__ uint32_t rows[THREADS];
            __shared__ uint64_t outs[THREADS];
            const uint32_t token0 = p.slices ? blockIdx.x / p.slices : blockIdx.x * p.perBlock;
            const uint32_t here   = p.slices ? 1u : min(p.perBlock, p.t.count - token0);
            grid_dependency_wait();
            grid_launch_dependents();
            if(threadIdx.x < here)
            {
                uint32_t outer, inner;
                rows[threadIdx.x] = rowOf(p.t, token0 + threadIdx.x, outer, inner);
                outs[threadIdx.x] = uint64_t(outer) * p.outOuter + uint64_t(inner) * p.outInner;
            }
            __syncthreads();
            auto get = [&](uint32_t row, uint32_t piece) {
                return loadPiece<T, V>(static_cast<T const*>(p.table) + uint64_t(row) * p.ldt + uint64_t(piece) * V);
            };
            auto put = [&](uint32_t t, uint32_t row, uint32_t piece, Piece<T, V> const& v) {
                Piece<OutT, V> o;
                if(row == NO_ROW)
                {
#pragma unroll
                    for(int i = 0; i < V; ++i)
                        o.v[i] = OutT(0.0f);
                }
                else if(std::is_same<T, OutT>::value && p.scale == 1.0f)
                    memcpy(&o, &v, sizeof(o)); // (65536 x 26 x 128 f16: 88 us with the conversions, 83 without)
                else
                {
#pragma unroll
                    for(int i = 0; i < V; ++i)
                        o.v[i] = fromFloat<OutT>(toFloat(v.v[i]) * p.scale);
                }
                storePiece<OutT, V>(static_cast<OutT*>(p.out) + outs[t] + uint64_t(piece) * V, o);
            };
            if(p.slices)
            {
                const uint32_t first = (blockIdx.x % p.slices) * (THREADS * U) + threadIdx.x, row = rows[0];
                Piece<T, V>    v[U];
#pragma unroll
                for(uint32_t u = 0; u < U; ++u)
                    if(row != NO_ROW && first + u * THREADS < p.pieces)
                        v[u] = get(row, first + u * THREADS);
#pragma unroll
                for(uint32_t u = 0; u < U; ++u)
                    if(first + u * THREADS < p.pieces)
                        put(0, row, first + u * THREADS, v[u]);
                return;
            }
            const uint32_t lanes = 1u << p.lanesLog2, step = THREADS >> p.lanesLog2;
            for(uint32_t piece = threadIdx.x & (lanes - 1u); piece < p.pieces; piece += lanes)
                for(uint32_t t0 = threadIdx.x >> p.lanesLog2; t0 < here; t0 += U * step)
                {
                    Piece<T, V> v[U];
                    uint32_t    row[U];
#pragma unroll
                    for(uint32_t u = 0; u < U; ++u)
                    {
                        row[u] = t0 + u * step < here ? rows[t0 + u * step] : NO_ROW;
                        if(row[u] != NO_ROW)
                            v[u] = get(row[u], piece);
                    }
#pragma unroll
                    for(uint32_t u = 0; u < U; ++u)
                        if(t0 + u * step < here)
                            put(t0 + u * step, row[u], piece, v[u]);
                }
        }

        // ---- clearing rows without a token -------------------------------------------------
        struct ClearParams
        {
            void*    table;
            uint64_t ldt;
            uint32_t pieces, lanesLog2; // of a row
            uint32_t blocks; // that clear, behind the others; 0: nothing to clear
            uint32_t rows, rowsPerBlock;
        };

        // The rows of [begin, end) that keep(row) does not name, by the calling block.
        template <typename OutT, int V, typename Keep>
        __device__ inline void clearRows(ClearParams const& c, uint64_t begin, uint64_t end, Keep keep)
        {
            const uint32_t lanes = 1u << c.lanesLog2;
            Piece<OutT, V> zero;
#pragma unroll
            for(int i = 0; i < V; ++i)
                zero.v[i] = OutT(0.0f);
            for(uint64_t row = begin + (threadIdx.x >> c.lanesLog2); row < end; row += blockDim.x >> c.lanesLog2)
                if(!keep(row))
                    for(uint32_t piece = threadIdx.x & (lanes - 1u); piece < c.pieces; piece += lanes)
                        storePiece<OutT, V>(static_cast<OutT*>(c.table) + row * c.ldt + uint64_t(piece) * V, zero);
        }

        // Digits of eight, nine or ten bits: two passes for tables of up to a million rows.
        template <uint32_t BITS>
        __device__ inline uint32_t digitOf(uint32_t key, uint32_t pass)
        {
            return (key >> (BITS * pass)) & ((1u << BITS) - 1u);
        }
        // Lanes of the warp with the same digit, among those that are `in`.  (A ballot for each bit:
        // match.any took most of the scattering kernel's time.)
        template <uint32_t BITS>
        __device__ inline uint32_t sameDigit(uint32_t digit, bool in)
        {
            uint32_t same = __ballot_sync(0xffffffffu, in);
#pragma unroll
            for(uint32_t b = 0; b < BITS; ++b)
            {
                const bool     set  = (digit >> b) & 1u;
                const uint32_t vote = __ballot_sync(0xffffffffu, set);
                same &= set ? vote : ~vote;
            }
            return same;
        }

        // ---- sorting few tokens: one block --------------------------------------------------
        constexpr uint32_t SMALL_THREADS = 1024;
        constexpr uint32_t SMALL_ITEMS   = 16;
        constexpr uint32_t SMALL_TOKENS  = SMALL_THREADS * SMALL_ITEMS;
        // One block sorts up to SMALL_ALWAYS tokens, and more where there is so much table to clear for each
        // that the other SMs have work beside it.  Whole calls, bf16 to f32, this way and the other:
        //     rows x dim      tokens   us                rows x dim      tokens   us
        //     50000 x 32          16   11.7  13.2        100000 x 16       4096   23.5  38.3
        //     50000 x 32        4096   23.4  20.2        2000000 x 32     16384   56    70
        //     32768 x 512         64   17.1  21.2        32768 x 512       4096   26.4  24.7
        //     1000 x 128        1024   13.9  10.4        1000 x 128        4096   17.6  11.7
        //     50000 x 128       1024   20.5  15.1        32768 x 4096     16384   131   115
        // So it is a coarse rule: right for narrow rows and for few tokens of a long table; for wide rows
        // the other way, whose search for rows without a token has become faster since, takes less
        // from some hundred tokens on, and always where the table has one digit of rows.
        constexpr uint32_t SMALL_ALWAYS      = 4096;
        constexpr uint64_t SMALL_CLEAR_BYTES = 12288; // of the table, a token
        constexpr uint32_t SMALL_WARPS   = SMALL_THREADS / 32;
        constexpr uint32_t SORT_BITS     = 10; // of a digit, at most
        constexpr uint32_t SORT_RADIX    = 1u << SORT_BITS;
        constexpr uint32_t CLEAR_BITS    = 65536; // rows that a clearing block looks over at a time
        template <uint32_t BITS>
        struct SmallShared
        {
            uint32_t keys[SMALL_TOKENS];
            uint32_t sums[SMALL_WARPS];
            uint16_t bins[SMALL_WARPS][1u << BITS];
            uint16_t tokens[SMALL_TOKENS];
        };
        static_assert(CLEAR_BITS / 8 <= SMALL_TOKENS * 4, "the clearing blocks' bits take the keys' place");

        // Block 0 sorts all tokens in shared memory; the others clear a share of the rows each, for
        // which they look through the tokens themselves.  (16384 tokens, 395 MB to clear: 75 us, 5.3 TB/s.)
        template <typename OutT, int V, uint32_t BITS>
        __global__ void __launch_bounds__(SMALL_THREADS)
            sortSmallKernel(const Tokens t, const ClearParams c, const uint32_t passes, uint2* sorted)
        {
            extern __shared__ uint8_t smem[];
            auto*          sh   = reinterpret_cast<SmallShared<BITS>*>(smem);
            const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
            grid_dependency_wait();
            grid_launch_dependents();
            uint32_t outer, inner;
            if(blockIdx.x > 0u)
            {
                const uint64_t begin = uint64_t(blockIdx.x - 1u) * t.rows / c.blocks;
                const uint64_t end   = uint64_t(blockIdx.x) * t.rows / c.blocks;
                for(uint64_t r0 = begin; r0 < end; r0 += CLEAR_BITS)
                {
                    const uint32_t count = uint32_t(min(uint64_t(CLEAR_BITS), end - r0));
                    __syncthreads();
                    for(uint32_t i = threadIdx.x; i < (count + 31u) / 32u; i += SMALL_THREADS)
                        sh->keys[i] = 0;
                    __syncthreads();
                    for(uint32_t i = threadIdx.x; i < t.count; i += SMALL_THREADS)
                    {
                        const uint32_t row = rowOf(t, i, outer, inner);
                        if(row >= r0 && row - r0 < count)
                            atomicOr(&sh->keys[uint32_t(row - r0) / 32u], 1u << (row - r0) % 32u);
                    }
                    __syncthreads();
                    clearRows<OutT, V>(c, r0, r0 + count, [&](uint64_t row) {
                        const uint32_t i = uint32_t(row - r0);
                        return (sh->keys[i / 32u] >> (i % 32u)) & 1u;
                    });
                }
                return;
            }
            // A warp's keys are neighbours, 32 of them a step.  A key's token and its rank among the
            // warp's keys of its digit share a register.
            constexpr uint32_t RADIX = 1u << BITS;
            static_assert(RADIX <= SMALL_THREADS, "a thread has a digit");
            const uint32_t items = (t.count + SMALL_THREADS - 1u) / SMALL_THREADS;
            const uint32_t warps = (t.count + 32u * items - 1u) / (32u * items); // that have keys
            const uint32_t first = warp * 32u * items + lane;
            uint32_t       key[SMALL_ITEMS], token[SMALL_ITEMS]; // rank << 16 | token
            {
                int64_t id[SMALL_ITEMS];
#pragma unroll
                for(uint32_t i = 0; i < SMALL_ITEMS; ++i)
                {
                    const uint32_t at = first + i * 32u;
                    id[i]             = i < items && at < t.count ? idOf(t, at, outer, token[i]) : -1;
                }
#pragma unroll
                for(uint32_t i = 0; i < SMALL_ITEMS; ++i)
                {
                    const uint32_t row = i < items && first + i * 32u < t.count ? rowOf(t, id[i], token[i]) : NO_ROW;
                    key[i]             = row == NO_ROW ? t.rows : row; // behind every row
                    token[i]           = first + i * 32u;
                }
            }
            for(uint32_t pass = 0; pass < passes; ++pass)
            {
                for(uint32_t i = threadIdx.x; i < warps * (RADIX / 2u); i += SMALL_THREADS)
                    reinterpret_cast<uint32_t*>(sh->bins)[i] = 0;
                __syncthreads();
                if(warp < warps)
                {
#pragma unroll
                    for(uint32_t i = 0; i < SMALL_ITEMS; ++i)
                        if(i < items)
                        {
                            const bool     in    = first + i * 32u < t.count;
                            const uint32_t d     = digitOf<BITS>(key[i], pass);
                            const uint32_t peers = sameDigit<BITS>(d, in);
                            const uint32_t rank  = sh->bins[warp][d] + __popc(peers & ((1u << lane) - 1u));
                            token[i]             = rank << 16 | (token[i] & 0xffffu);
                            __syncwarp();
                            if(in && (peers >> lane) == 1u) // the last of its digit
                                sh->bins[warp][d] = uint16_t(rank + 1u);
                            __syncwarp();
                        }
                }
                __syncthreads();
                // thread = digit: where the keys of each warp go
                uint32_t sum = 0;
                if(threadIdx.x < RADIX)
#pragma unroll 8
                    for(uint32_t w = 0; w < warps; ++w)
                        sum += sh->bins[w][threadIdx.x];
                uint32_t before = sum;
#pragma unroll
                for(uint32_t d = 1; d < 32u; d *= 2u)
                {
                    const uint32_t other = __shfl_up_sync(0xffffffffu, before, d);
                    if(lane >= d)
                        before += other;
                }
                if(lane == 31u)
                    sh->sums[warp] = before;
                before -= sum;
                __syncthreads();
                if(threadIdx.x < RADIX)
                {
                    for(uint32_t w = 0; w < warp; ++w)
                        before += sh->sums[w];
#pragma unroll 8
                    for(uint32_t w = 0; w < warps; ++w)
                    {
                        const uint32_t count     = sh->bins[w][threadIdx.x];
                        sh->bins[w][threadIdx.x] = uint16_t(before);
                        before += count;
                    }
                }
                __syncthreads();
                const bool last = pass + 1u == passes;
#pragma unroll
                for(uint32_t i = 0; i < SMALL_ITEMS; ++i)
                    if(i < items && first + i * 32u < t.count)
                    {
                        const uint32_t to = sh->bins[warp][digitOf<BITS>(key[i], pass)] + (token[i] >> 16);
                        if(last)
                            sorted[to] = make_uint2(key[i], token[i] & 0xffffu);
                        else
                        {
                            sh->keys[to]   = key[i];
                            sh->tokens[to] = uint16_t(token[i]);
                        }
                    }
                if(last)
                    break;
                __syncthreads();
#pragma unroll
                for(uint32_t i = 0; i < SMALL_ITEMS; ++i)
                    if(i < items && first + i * 32u < t.count)
                    {
                        key[i]   = sh->keys[first + i * 32u];
                        token[i] = sh->tokens[first + i * 32u];
                    }
            }
        }

        // ---- sorting many tokens -------------------------------------------------------------
        // A block has a tile of THREADS x ITEMS keys.  Four a thread make the blocks that hide a block's
        // own latency, sixteen write longer stretches and leave fewer counts to add up: whole calls
        // take 57 us with four and 61 with sixteen at 200000 tokens, 160 and 161 at 1.7 million, 292
        // and 264 at four million.
        // Up to FEW_TILES tiles, the scattering blocks add up the tiles' counts themselves instead of
        // a kernel of its own: 32.8 us so and 35.6 with the kernel at 20 tiles, 41.2 and 42.6 at 59,
        // 47.4 and 44.2 at 79.
        constexpr uint32_t SORT_WARPS = THREADS / 32;
        constexpr uint32_t FEW_ITEMS = 4, MANY_ITEMS = 16, MANY_TOKENS = 2000000, FEW_TILES = 64;

        // bins[digit] = keys of the tile
        template <uint32_t ITEMS, uint32_t BITS>
        __device__ inline void countDigits(uint32_t* bins, uint32_t const (&key)[ITEMS], uint32_t first, uint32_t n,
                                           uint32_t pass, uint32_t* counts)
        {
            constexpr uint32_t radix = 1u << BITS;
            for(uint32_t d = threadIdx.x; d < radix; d += THREADS)
                bins[d] = 0;
            __syncthreads();
#pragma unroll
            for(uint32_t i = 0; i < ITEMS; ++i)
            {
                // one addition for the equal digits of a warp: a hot row would queue 32
                const bool     in    = uint64_t(first) + i * THREADS < n;
                const uint32_t digit = digitOf<BITS>(key[i], pass);
                const uint32_t peers = sameDigit<BITS>(digit, in);
                if(in && (peers & ((1u << (threadIdx.x % 32u)) - 1u)) == 0u)
                    atomicAdd(&bins[digit], uint32_t(__popc(peers)));
            }
            __syncthreads();
            for(uint32_t d = threadIdx.x; d < radix; d += THREADS)
                counts[uint64_t(blockIdx.x) * radix + d] = bins[d];
        }

        // Row of every token, and the first digit's counts[tile][digit].
        template <uint32_t ITEMS, uint32_t BITS>
        __global__ void __launch_bounds__(THREADS) keysKernel(const Tokens t, uint32_t* keys, uint32_t* counts)
        {
            __shared__ uint32_t bins[1u << BITS];
            grid_dependency_wait();
            grid_launch_dependents();
            const uint32_t first = blockIdx.x * (THREADS * ITEMS) + threadIdx.x;
            uint32_t       key[ITEMS], outer, inner[ITEMS];
            int64_t        id[ITEMS];
#pragma unroll
            for(uint32_t i = 0; i < ITEMS; ++i)
            {
                const uint32_t token = first + i * THREADS;
                id[i]                = token < t.count ? idOf(t, token, outer, inner[i]) : -1;
            }
#pragma unroll
            for(uint32_t i = 0; i < ITEMS; ++i)
            {
                const uint32_t token = first + i * THREADS;
                key[i]               = t.rows; // behind every row
                if(token < t.count)
                {
                    const uint32_t row = rowOf(t, id[i], inner[i]);
                    if(row != NO_ROW)
                        key[i] = row;
                    keys[token] = key[i];
                }
            }
            countDigits<ITEMS, BITS>(bins, key, first, t.count, 0, counts);
        }

        template <uint32_t ITEMS, uint32_t BITS>
        __global__ void __launch_bounds__(THREADS)
            countKernel(uint2 const* pairs, uint32_t n, uint32_t pass, uint32_t* counts)
        {
            __shared__ uint32_t bins[1u << BITS];
            grid_dependency_wait();
            grid_launch_dependents();
            const uint32_t first = blockIdx.x * (THREADS * ITEMS) + threadIdx.x;
            uint32_t       key[ITEMS];
#pragma unroll
            for(uint32_t i = 0; i < ITEMS; ++i)
                key[i] = first + i * THREADS < n ? pairs[first + i * THREADS].x : 0u;
            countDigits<ITEMS, BITS>(bins, key, first, n, pass, counts);
        }

        // Exclusive sum of a value over the block's threads, and the total.
        __device__ inline uint32_t blockScan(uint32_t v, uint32_t* warps, uint32_t& total)
        {
            const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
            uint32_t       sum = v;
#pragma unroll
            for(uint32_t d = 1; d < 32u; d *= 2u)
            {
                const uint32_t other = __shfl_up_sync(0xffffffffu, sum, d);
                if(lane >= d)
                    sum += other;
            }
            __syncthreads();
            if(lane == 31u)
                warps[warp] = sum;
            __syncthreads();
            uint32_t before = 0;
            total           = 0;
#pragma unroll
            for(uint32_t w = 0; w < SORT_WARPS; ++w)
            {
                before += w < warp ? warps[w] : 0u;
                total += warps[w];
            }
            return before + sum - v;
        }

        // A block has eight digits, a sector of each tile's counts: they become exclusive sums over the
        // tiles, their totals go to totals[digit].  Four times 32 groups of eight threads have a
        // stretch of tiles each.
        constexpr uint32_t SCAN_THREADS = 1024, SCAN_DIGITS = 8;
        __global__ void __launch_bounds__(SCAN_THREADS) scanKernel(uint32_t* counts, uint32_t tiles, uint32_t radix, uint32_t* totals)
        {
            constexpr uint32_t GROUPS = SCAN_THREADS / SCAN_DIGITS;
            __shared__ uint32_t sums[32][SCAN_DIGITS];
            grid_dependency_wait();
            grid_launch_dependents();
            const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, column = threadIdx.x % SCAN_DIGITS;
            const uint32_t group = threadIdx.x / SCAN_DIGITS, digit = blockIdx.x * SCAN_DIGITS + column;
            const uint32_t begin = uint32_t(uint64_t(tiles) * group / GROUPS), end = uint32_t(uint64_t(tiles) * (group + 1u) / GROUPS);
            const bool     in    = digit < radix;
            uint32_t       sum   = 0;
#pragma unroll 8
            for(uint32_t t = begin; t < end; ++t)
                sum += in ? counts[uint64_t(t) * radix + digit] : 0u;
            uint32_t upTo = sum; // over the warp's groups so far
#pragma unroll
            for(uint32_t d = SCAN_DIGITS; d < 32u; d *= 2u)
            {
                const uint32_t other = __shfl_up_sync(0xffffffffu, upTo, d);
                if(lane >= d)
                    upTo += other;
            }
            if(lane >= 32u - SCAN_DIGITS)
                sums[warp][column] = upTo;
            __syncthreads();
            uint32_t before = upTo - sum, total = 0;
#pragma unroll
            for(uint32_t w = 0; w < 32u; ++w)
            {
                before += w < warp ? sums[w][column] : 0u;
                total += sums[w][column];
            }
            if(!in)
                return;
            constexpr uint32_t BATCH = 8; // loaded together
            for(uint32_t t0 = begin; t0 < end; t0 += BATCH)
            {
                uint32_t count[BATCH];
#pragma unroll
                for(uint32_t i = 0; i < BATCH; ++i)
                    count[i] = t0 + i < end ? counts[uint64_t(t0 + i) * radix + digit] : 0u;
#pragma unroll
                for(uint32_t i = 0; i < BATCH; ++i)
                {
                    if(t0 + i < end)
                        counts[uint64_t(t0 + i) * radix + digit] = before;
                    before += count[i];
                }
            }
            if(group == 0u)
                totals[digit] = total;
        }

        // Moves every key of a tile, with its token, to its place among the keys of this digit:
        // those of smaller digits, of earlier tiles, of earlier warps, of earlier rows of 32 and
        // of smaller lanes come first.  The tile is put in order in shared memory first, so that
        // neighbouring threads write neighbouring places.  pairs == nullptr: the first pass, key i
        // of `keys` belongs to token i.
        template <uint32_t ITEMS, uint32_t BITS>
        struct ScatterShared
        {
            uint2    tile[THREADS * ITEMS];
            uint16_t bins[SORT_WARPS][1u << BITS];
            uint32_t shifts[1u << BITS]; // place of a digit's keys minus their place in the tile
            uint32_t warps[SORT_WARPS];
        };

        template <uint32_t ITEMS, uint32_t BITS>
        __global__ void __launch_bounds__(THREADS, 3)
            scatterKernel(uint32_t const* keys, uint2 const* pairs, uint32_t n, uint32_t pass, uint32_t tiles,
                          uint32_t const* counts, uint32_t const* totals, uint2* out)
        {
            constexpr uint32_t RADIX = 1u << BITS, PER = RADIX / THREADS; // digits of a thread
            extern __shared__ uint8_t smem[];
            auto*          sh   = reinterpret_cast<ScatterShared<ITEMS, BITS>*>(smem);
            const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
            grid_dependency_wait();
            grid_launch_dependents();
            for(uint32_t i = threadIdx.x; i < SORT_WARPS * RADIX / 2u; i += THREADS)
                reinterpret_cast<uint32_t*>(sh->bins)[i] = 0;
            __syncthreads();
            const uint32_t tile0 = blockIdx.x * (THREADS * ITEMS), here = min(THREADS * ITEMS, n - tile0);
            const uint32_t first = warp * (32u * ITEMS) + lane;
            uint2          pair[ITEMS];
            uint32_t       rank[ITEMS];
#pragma unroll
            for(uint32_t i = 0; i < ITEMS; ++i)
            {
                const uint32_t at = first + i * 32u;
                pair[i]           = make_uint2(0u, tile0 + at);
                if(at < here)
                {
                    if(pairs)
                        pair[i] = pairs[tile0 + at];
                    else
                        pair[i].x = keys[tile0 + at];
                }
            }
#pragma unroll
            for(uint32_t i = 0; i < ITEMS; ++i)
            {
                const bool     in    = first + i * 32u < here;
                const uint32_t d     = digitOf<BITS>(pair[i].x, pass);
                const uint32_t peers = sameDigit<BITS>(d, in);
                rank[i]              = (in ? sh->bins[warp][d] : 0u) + __popc(peers & ((1u << lane) - 1u));
                __syncwarp();
                if(in && (peers >> lane) == 1u) // the last of its digit
                    sh->bins[warp][d] = uint16_t(rank[i] + 1u);
                __syncwarp();
            }
            __syncthreads();
            // thread = neighbouring digits: where the keys of each warp go in the tile, and the tile's
            // in the whole
            {
                const uint32_t d0 = threadIdx.x * PER;
                uint32_t       sums[PER], all[PER], earlier[PER], total, mine = 0, whole = 0;
                if(tiles != 0u)
                {
                    // few tiles: their counts are added up here instead of by a kernel of its own
#pragma unroll
                    for(uint32_t j = 0; j < PER; ++j)
                        all[j] = earlier[j] = 0;
#pragma unroll 8
                    for(uint32_t t = 0; t < tiles; ++t)
#pragma unroll
                        for(uint32_t j = 0; j < PER; ++j)
                        {
                            const uint32_t count = counts[uint64_t(t) * RADIX + d0 + j];
                            all[j] += count;
                            earlier[j] += t < blockIdx.x ? count : 0u;
                        }
                }
                else
                {
#pragma unroll
                    for(uint32_t j = 0; j < PER; ++j)
                    {
                        all[j]     = totals[d0 + j];
                        earlier[j] = counts[uint64_t(blockIdx.x) * RADIX + d0 + j];
                    }
                }
#pragma unroll
                for(uint32_t j = 0; j < PER; ++j)
                {
                    sums[j] = 0;
#pragma unroll
                    for(uint32_t w = 0; w < SORT_WARPS; ++w)
                        sums[j] += sh->bins[w][d0 + j];
                    mine += sums[j];
                    whole += all[j];
                }
                uint32_t local  = blockScan(mine, sh->warps, total);
                uint32_t global = blockScan(whole, sh->warps, total);
#pragma unroll
                for(uint32_t j = 0; j < PER; ++j)
                {
                    uint32_t at = local;
#pragma unroll
                    for(uint32_t w = 0; w < SORT_WARPS; ++w)
                    {
                        const uint32_t count = sh->bins[w][d0 + j];
                        sh->bins[w][d0 + j]  = uint16_t(at);
                        at += count;
                    }
                    sh->shifts[d0 + j] = global + earlier[j] - local;
                    local += sums[j];
                    global += all[j];
                }
            }
            __syncthreads();
#pragma unroll
            for(uint32_t i = 0; i < ITEMS; ++i)
                if(first + i * 32u < here)
                    sh->tile[sh->bins[warp][digitOf<BITS>(pair[i].x, pass)] + rank[i]] = pair[i];
            __syncthreads();
            for(uint32_t i = threadIdx.x; i < here; i += THREADS)
            {
                const uint2 p = sh->tile[i];
                out[sh->shifts[digitOf<BITS>(p.x, pass)] + i] = p;
            }
        }

        // ---- summing runs ------------------------------------------------------------------
        constexpr uint32_t SUM_ITEMS = 1024; // of a block
        constexpr uint32_t RING_BYTES = 128; // of a thread: pieces on their way
        struct SumParams
        {
            uint2 const* sorted; // (row, token), equal rows next to each other
            void const*  grad;
            uint64_t     gradOuter, gradInner;
            Divisor      inner;
            uint32_t     n, chunk, parts, rows; // parts: blocks' worth of chunks
            uint32_t     pieces, lanesLog2, slices; // pieces of a row; threads side by side on it; blocks
            uint32_t     blocks; // that sum; those behind them clear
            void*        table;
            uint64_t     ldt;
            float        scale;
            uint32_t     accumulate;
            uint32_t*    pieceKeys; // two of each part: run from the left, run to the right; nullptr: one part
            float*       pieceSums; // rows of `pieces * V`
        };

        // A finished row's piece.
        template <typename OutT, int V>
        __device__ inline void finishRow(SumParams const& p, uint32_t row, uint32_t piece, float const (&sum)[V])
        {
            OutT*          at = static_cast<OutT*>(p.table) + uint64_t(row) * p.ldt + uint64_t(piece) * V;
            Piece<OutT, V> o;
            if(p.accumulate)
            {
                o = loadPiece<OutT, V>(at);
#pragma unroll
                for(int i = 0; i < V; ++i)
                    o.v[i] = fromFloat<OutT>(fmaf(sum[i], p.scale, toFloat(o.v[i])));
            }
            else
            {
#pragma unroll
                for(int i = 0; i < V; ++i)
                    o.v[i] = fromFloat<OutT>(sum[i] * p.scale);
            }
            storePiece<OutT, V>(at, o);
        }

        // First of the n sorted items whose row is not below `row`.  Seven items are looked at together:
        // the search is a chain of waits for memory, and three bits a link make it a third as long.
        // (38000 tokens of 300 rows of 8: the kernel took 23 us with one item at a time, 10 so.)
        __device__ inline uint32_t lowerBound(uint2 const* sorted, uint32_t n, uint64_t row)
        {
            uint32_t low = 0, high = n;
            while(low < high)
            {
                uint32_t at[7];
#pragma unroll
                for(uint32_t i = 0; i < 7u; ++i)
                    at[i] = low + uint32_t(uint64_t(high - low) * (i + 1u) / 8u); // < high
                bool less[7];
#pragma unroll
                for(uint32_t i = 0; i < 7u; ++i)
                    less[i] = sorted[at[i]].x < row;
#pragma unroll
                for(uint32_t i = 0; i < 7u; ++i) // behind the last one that is below
                    low = less[i] ? at[i] + 1u : low;
#pragma unroll
                for(uint32_t i = 7; i-- > 0u;) // up to the first one that is not
                    high = less[i] ? high : at[i];
            }
            return low;
        }

        // A thread's ring of pieces that cp.async brings: nobody else reads them, so there is nothing to
        // synchronise, and the loads hold no registers while they fly.  (With the pieces of eight
        // items in registers the kernel ran 512 threads to an SM and 2.3 TB/s.)
        template <typename T, int V>
        struct Ring
        {
            // (single 16-bit values travel in the aligned word that holds them)
            static constexpr uint32_t BYTES = sizeof(T) * V < 4 ? 4 : sizeof(T) * V; // 4, 8 or 16: a copy
            static constexpr uint32_t DEPTH = RING_BYTES / BYTES > 16 ? 16 : RING_BYTES / BYTES;

            // slot s of the calling thread; the threads of a block lie side by side
            static __device__ uint8_t* at(uint8_t* ring, uint32_t s)
            {
                return ring + (s * blockDim.x + threadIdx.x) * BYTES;
            }
            static __device__ void load(uint8_t* ring, uint32_t s, T const* from)
            {
                uint64_t src = reinterpret_cast<uint64_t>(from);
                if constexpr(sizeof(T) * V < 4)
                    src &= ~uint64_t(3);
                const uint32_t to = uint32_t(__cvta_generic_to_shared(at(ring, s)));
                if constexpr(BYTES == 16) // past L1, which has no use for them
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
                else
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(src), "n"(BYTES) : "memory");
            }
            static __device__ Piece<T, V> get(uint8_t* ring, uint32_t s, uint64_t place)
            {
                Piece<T, V> p;
                if constexpr(sizeof(T) * V < 4)
                    p.v[0] = reinterpret_cast<T const*>(at(ring, s))[place / sizeof(T) % 2u];
                else
                    p = *reinterpret_cast<Piece<T, V> const*>(at(ring, s));
                return p;
            }
        };

        // Threads side by side share a chunk of items, one piece of the row each.  The block puts
        // its items' rows and places into shared memory first, so that no load waits for another.
        // (65536 x 26 x 128 f16 to f32: 95 us, 5.0 TB/s, reading rows of 256 bytes in the table's order.)
        template <typename T, typename OutT, int V>
        __global__ void __launch_bounds__(THREADS) sumKernel(const SumParams p, const ClearParams c)
        {
            using R = Ring<T, V>;
            __shared__ uint32_t rows[SUM_ITEMS + 2]; // of the items, and one on each side
            __shared__ uint64_t places[SUM_ITEMS + 2]; // of their gradients, in elements
            extern __shared__ uint4 ringWords[]; // R::DEPTH * R::BYTES of each thread
            uint8_t* const ring = reinterpret_cast<uint8_t*>(ringWords);
            grid_dependency_wait();
            grid_launch_dependents();
            if(blockIdx.x >= p.blocks)
            {
                const uint64_t begin = uint64_t(blockIdx.x - p.blocks) * c.rowsPerBlock;
                const uint64_t end   = min(uint64_t(c.rows), begin + c.rowsPerBlock);
                for(uint32_t i = threadIdx.x; i < uint32_t(end - begin); i += blockDim.x)
                {
                    const uint32_t at = lowerBound(p.sorted, p.n, begin + i);
                    rows[i]           = at < p.n && p.sorted[at].x == begin + i;
                }
                __syncthreads();
                return clearRows<OutT, V>(c, begin, end, [&](uint64_t row) { return rows[row - begin] != 0u; });
            }
            const uint32_t lanes = 1u << p.lanesLog2, groups = blockDim.x >> p.lanesLog2;
            const uint32_t slice = blockIdx.x % p.slices;
            const uint64_t item0 = uint64_t(blockIdx.x / p.slices) * groups * p.chunk;
            for(uint32_t i = threadIdx.x; i < groups * p.chunk + 2u; i += blockDim.x)
            {
                const uint64_t at   = item0 + i; // of item at - 1
                const uint2    pair = at >= 1u && at <= p.n ? p.sorted[at - 1u] : make_uint2(NO_ROW, 0u);
                uint32_t       outer = pair.y, in = 0;
                if(p.inner.d > 1u)
                {
                    outer = p.inner.of(pair.y);
                    in    = pair.y - outer * p.inner.d;
                }
                rows[i]   = pair.x;
                places[i] = uint64_t(outer) * p.gradOuter + uint64_t(in) * p.gradInner;
            }
            __syncthreads();
            const uint32_t piece = slice * lanes + (threadIdx.x & (lanes - 1u));
            const uint32_t local = (threadIdx.x >> p.lanesLog2) * p.chunk; // first item in shared memory
            const uint64_t begin = item0 + local;
            const uint32_t count = piece < p.pieces && begin < p.n ? uint32_t(min(uint64_t(p.chunk), p.n - begin)) : 0u;
            const uint32_t  before = rows[local], after = rows[local + count + 1u];
            uint32_t const* rowAt  = rows + local + 1u;
            uint64_t const* place  = places + local + 1u;
            T const*        grad   = static_cast<T const*>(p.grad) + uint64_t(piece) * V;

            float    sum[V], left[V]; // of the current run; of the one that came from the left
            uint32_t run      = NO_ROW; // row of the current run
            bool     fromLeft = false;
            uint32_t leftKey = NO_ROW, rightKey = NO_ROW;
#pragma unroll
            for(int j = 0; j < V; ++j)
                sum[j] = left[j] = 0.0f;
            auto load = [&](uint32_t i) {
                if(i < count && rowAt[i] < p.rows)
                    R::load(ring, i % R::DEPTH, grad + place[i]);
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll
            for(uint32_t i = 0; i < R::DEPTH; ++i)
                load(i);
            for(uint32_t i = 0;; ++i)
            {
                const uint32_t row = i < count ? rowAt[i] : NO_ROW;
                if(row != run || i == count)
                {
                    // the end of a run
                    if(run < p.rows)
                    {
                        const bool toRight = i == count && after == run;
                        if(!fromLeft && !toRight)
                            finishRow<OutT, V>(p, run, piece, sum);
                        else
                        {
                            if(fromLeft)
                            {
                                leftKey = run;
#pragma unroll
                                for(int j = 0; j < V; ++j)
                                    left[j] = sum[j];
                            }
                            if(toRight) // a piece of a run that starts here, or one that passes through
                                rightKey = run | (fromLeft ? PASSES : 0u);
                        }
                    }
                    if(i == count)
                        break;
                    run      = row;
                    fromLeft = i == 0u && before == row;
#pragma unroll
                    for(int j = 0; j < V; ++j)
                        sum[j] = 0.0f;
                }
                asm volatile("cp.async.wait_group %0;" ::"n"(R::DEPTH - 1) : "memory");
                if(row < p.rows)
                {
                    const Piece<T, V> v = R::get(ring, i % R::DEPTH, sizeof(T) * V < 4 ? reinterpret_cast<uint64_t>(grad + place[i]) : 0u);
#pragma unroll
                    for(int j = 0; j < V; ++j)
                        sum[j] += toFloat(v.v[j]);
                }
                load(i + R::DEPTH);
            }
            // The runs that cross the block's chunks: the pieces take the rings' place.
            __shared__ uint32_t leftKeys[32], rightKeys[32], ends[2];
            const uint32_t group = threadIdx.x >> p.lanesLog2, lane = threadIdx.x & (lanes - 1u);
            auto           pieceAt = [&](uint32_t g, uint32_t side) {
                return reinterpret_cast<float*>(ringWords) + ((2u * g + side) * lanes + lane) * V;
            };
            __syncthreads();
            if(lane == 0u)
            {
                leftKeys[group]  = leftKey;
                rightKeys[group] = rightKey;
            }
            if(threadIdx.x < 2u)
                ends[threadIdx.x] = NO_ROW;
            if(leftKey < p.rows)
            {
#pragma unroll
                for(int j = 0; j < V; ++j)
                    pieceAt(group, 0)[j] = left[j];
            }
            if(rightKey < p.rows)
            {
#pragma unroll
                for(int j = 0; j < V; ++j)
                    pieceAt(group, 1)[j] = sum[j];
            }
            __syncthreads();
            const uint64_t part = blockIdx.x / p.slices, width = uint64_t(p.pieces) * V;
            // the run `row` whose piece of chunk g, on its `side`, comes first in the block
            auto follow = [&](uint32_t row, uint32_t g, uint32_t side) {
#pragma unroll
                for(int j = 0; j < V; ++j)
                    sum[j] = pieceAt(g, side)[j];
                bool on = side == 1u || rightKeys[g] == (row | PASSES);
                for(++g; on && g < groups; ++g)
                {
#pragma unroll
                    for(int j = 0; j < V; ++j)
                        sum[j] += pieceAt(g, 0)[j];
                    on = rightKeys[g] == (row | PASSES);
                }
                if(side == 1u && !on)
                {
                    if(piece < p.pieces)
                        finishRow<OutT, V>(p, row, piece, sum);
                    return;
                }
                if(lane == 0u)
                {
                    if(side == 0u)
                        ends[0] = row;
                    if(on)
                        ends[1] = row | (side == 0u ? PASSES : 0u);
                }
                if(piece < p.pieces)
                {
                    Piece<float, V> s;
#pragma unroll
                    for(int j = 0; j < V; ++j)
                        s.v[j] = sum[j];
                    storePiece<float, V>(p.pieceSums + (2u * part + side) * width + uint64_t(piece) * V, s);
                }
            };
            const uint32_t starts = rightKeys[group];
            if(starts < p.rows)
                follow(starts, group, 1);
            if(group == 0u && leftKeys[0] < p.rows)
                follow(leftKeys[0], 0, 0);
            if(!p.pieceKeys || slice != 0u)
                return;
            __syncthreads();
            if(threadIdx.x < 2u)
                p.pieceKeys[2u * part + threadIdx.x] = ends[threadIdx.x];
        }

        // Joins the runs that cross parts, as a block's worth of chunks is called.  A group of threads
        // side by side has a part: where a run starts there that goes on to the right, the row is the
        // sum of that piece, of those of the parts that the run passes through, and of the last one's,
        // in this order.  Runs of more than JOIN_FEW pieces are left to the whole block: its groups
        // take the pieces in turn.
        constexpr uint32_t JOIN_FEW = 16;

        template <typename OutT, int V>
        __global__ void __launch_bounds__(THREADS) joinKernel(const SumParams p)
        {
            constexpr uint32_t U = 4;
            __shared__ uint32_t longs[THREADS], longCount, end;
            __shared__ float    sums[THREADS][V + 1];
            if(threadIdx.x == 0u)
                longCount = 0;
            __syncthreads();
            grid_dependency_wait();
            grid_launch_dependents();
            const uint32_t lanes = 1u << p.lanesLog2, groups = THREADS >> p.lanesLog2;
            const uint32_t slice = blockIdx.x % p.slices;
            const uint32_t lane = threadIdx.x & (lanes - 1u), group = threadIdx.x >> p.lanesLog2;
            const uint32_t piece = slice * lanes + lane;
            const uint64_t width = uint64_t(p.pieces) * V;
            float const*   at    = p.pieceSums + uint64_t(piece) * V;
            auto           rightKey = [&](uint32_t c) { return p.pieceKeys[2u * uint64_t(c) + 1u]; };
            float          sum[V];
            // pieces begin, begin + step, ... of a run of `count` that starts in part `first`
            auto add = [&](uint32_t first, uint32_t begin, uint32_t count, uint32_t step) {
#pragma unroll
                for(int j = 0; j < V; ++j)
                    sum[j] = 0.0f;
                for(uint32_t i0 = begin; i0 < count; i0 += U * step)
                {
                    Piece<float, V> v[U];
#pragma unroll
                    for(uint32_t u = 0; u < U; ++u)
                    {
                        const uint32_t i = i0 + u * step;
                        if(i < count) // the first piece went to the right, the others come from the left
                            v[u] = loadPiece<float, V>(at + (2u * uint64_t(first + i) + (i == 0u ? 1u : 0u)) * width);
                    }
#pragma unroll
                    for(uint32_t u = 0; u < U; ++u)
                        if(i0 + u * step < count)
                        {
#pragma unroll
                            for(int j = 0; j < V; ++j)
                                sum[j] += v[u].v[j];
                        }
                }
            };
            const uint64_t mine = uint64_t(blockIdx.x / p.slices) * groups + group;
            if(mine + 1u < p.parts)
            {
                const uint32_t first = uint32_t(mine), row = rightKey(first);
                if(row < p.rows) // a run starts here and goes on
                {
                    uint32_t count = 2;
                    while(count <= JOIN_FEW && rightKey(first + count - 1u) == (row | PASSES))
                        ++count;
                    if(count > JOIN_FEW)
                    {
                        if(lane == 0u)
                            longs[atomicAdd(&longCount, 1u)] = first;
                    }
                    else if(piece < p.pieces)
                    {
                        add(first, 0, count, 1);
                        finishRow<OutT, V>(p, row, piece, sum);
                    }
                }
            }
            __syncthreads();
            for(uint32_t l = 0; l < longCount; ++l)
            {
                const uint32_t first = longs[l], row = rightKey(first);
                for(uint32_t c0 = first + 1u;; c0 += THREADS) // the run's last part
                {
                    __syncthreads();
                    if(threadIdx.x == 0u)
                        end = 0xffffffffu;
                    __syncthreads();
                    const uint32_t c = c0 + threadIdx.x;
                    if(c >= p.parts || rightKey(c) != (row | PASSES))
                        atomicMin(&end, c);
                    __syncthreads();
                    if(end != 0xffffffffu)
                        break;
                }
                const uint32_t count = end - first + 1u;
                if(piece < p.pieces)
                    add(first, group, count, groups);
#pragma unroll
                for(int j = 0; j < V; ++j)
                    sums[threadIdx.x][j] = sum[j];
                __syncthreads();
                if(group != 0u)
                    continue;
                for(uint32_t g = 1; g < groups && g < count; ++g)
                {
#pragma unroll
                    for(int j = 0; j < V; ++j)
                        sum[j] += sums[(g << p.lanesLog2) + threadIdx.x][j];
                }
                if(piece < p.pieces)
                    finishRow<OutT, V>(p, row, piece, sum);
            }
        }

        // ---- host side ---------------------------------------------------------------------
        bool valueType(int dtype)
        {
            return dtype == B200WMMA_F16 || dtype == B200WMMA_BF16 || dtype == B200WMMA_F32;
        }
        bool aligned(void const* p, uint64_t bytes)
        {
            return reinterpret_cast<uintptr_t>(p) % bytes == 0;
        }
        uint32_t log2Up(uint64_t v)
        {
            uint32_t l = 0;
            while((1ull << l) < v)
                ++l;
            return l;
        }
        // Threads side by side on a row.
        uint32_t rowLanesLog2(uint32_t pieces)
        {
            const uint32_t l = log2Up(pieces);
            return l > 8u ? 8u : l;
        }
        // Values of a piece: 8, 4, 2 or 1, whatever divides dim and keeps every piece of the given
        // tensors on its boundary.  `strides`: distances of rows, in elements.
        template <typename... Strides>
        uint32_t pieceSize(uint32_t dim, void const* base, uint64_t elem, uint32_t most, Strides... strides)
        {
            for(uint32_t v = most; v > 1u; v /= 2u)
            {
                const uint64_t bytes = v * elem;
                if(dim % v == 0u && aligned(base, bytes) && ((strides * elem % bytes == 0) && ...))
                    return v;
            }
            return 1;
        }

        // f(v) with v as a constant
        template <typename F>
        int withPiece(uint32_t v, F f)
        {
            switch(v)
            {
            case 8:
                return f(std::integral_constant<int, 8>());
            case 4:
                return f(std::integral_constant<int, 4>());
            case 2:
                return f(std::integral_constant<int, 2>());
            }
            return f(std::integral_constant<int, 1>());
        }

        template <typename T, typename OutT, int V>
        int lookup(LookupParams p, uint32_t dim, cudaStream_t stream)
        {
            p.pieces    = dim / V;
            p.lanesLog2 = rowLanesLog2(p.pieces);
            // Fewer threads side by side where that leaves fewer of them without a piece, down to those of a
            // line of 128 bytes (701000 rows of 82 f32, 41 pieces: 88 us with 64 threads to a row, 77 with
            // 16; 122000 rows of 247 bf16, 247 pieces: 50 us with 256, 242 with 8).
            auto rounded = [&](uint32_t lanes) { return (p.pieces + (1u << lanes) - 1u) >> lanes << lanes; };
            for(uint32_t l = p.lanesLog2; (V * sizeof(OutT)) << l >= 128u; --l)
                p.lanesLog2 = rounded(l) < rounded(p.lanesLog2) ? l : p.lanesLog2;
            // 4096 pieces to a block (16 a thread), but blocks for every SM first
            uint32_t per = p.pieces >= 4096u ? 1u : 4096u / p.pieces;
            per          = per > THREADS ? THREADS : per;
            const uint32_t spread = (p.t.count + 4u * 148u - 1u) / (4u * 148u);
            p.perBlock            = per < spread ? per : spread;
            p.slices              = 0;
            constexpr uint32_t U  = lookupUnroll(V);
            if(p.perBlock < U && p.pieces > THREADS)
            {
                p.perBlock = 1;
                p.slices   = (p.pieces + THREADS * U - 1u) / (THREADS * U);
            }
            const uint64_t blocks = (uint64_t(p.t.count) + p.perBlock - 1u) / p.perBlock * (p.slices ? p.slices : 1u);
            if(blocks > 0x7fffffffull)
                return B200WMMA_ERR_TOO_LARGE;
            return cudaToStatus(launchOverlapped(lookupKernel<T, OutT, V>, dim3(uint32_t(blocks)), dim3(THREADS), 0, stream, p));
        }

        template <typename T, typename OutT>
        int lookupTyped(LookupParams const& p, uint32_t dim, cudaStream_t stream)
        {
            const uint32_t v = pieceSize(dim, p.out, sizeof(OutT), pieceSize(dim, p.table, sizeof(T), 8, p.ldt), p.outOuter,
                                         p.outInner);
            return withPiece(v, [&](auto V) { return lookup<T, OutT, V.value>(p, dim, stream); });
        }

        template <typename T>
        int lookupFrom(int out, LookupParams const& p, uint32_t dim, cudaStream_t stream)
        {
            switch(out)
            {
            case B200WMMA_F16:
                return lookupTyped<T, __half>(p, dim, stream);
            case B200WMMA_BF16:
                return lookupTyped<T, __nv_bfloat16>(p, dim, stream);
            }
            return lookupTyped<T, float>(p, dim, stream);
        }

        // Threads of a block of the sum: sixteen rows side by side, a warp at least.
        uint32_t sumThreads(uint32_t lanesLog2)
        {
            return lanesLog2 == 0u ? 32u : lanesLog2 >= 4u ? THREADS : 16u << lanesLog2;
        }

        // Blocks along the tokens.
        uint64_t partsOf(uint32_t count, uint32_t chunk, uint32_t lanesLog2)
        {
            const uint64_t per = uint64_t(sumThreads(lanesLog2) >> lanesLog2) * chunk;
            return (count + per - 1u) / per;
        }

        // The workspace of the gradient; offsets in bytes.  The chunks go by the sizes alone.
        struct Plan
        {
            uint64_t keys, pairs[2], counts, totals, pieceKeys, pieceSums, bytes;
            uint32_t tiles, passes, digitBits, chunk;
            bool     small;
        };

        // Whether one block sorts: see SMALL_ALWAYS.  `clear`: bytes to be cleared, at most.
        bool sortsSmall(uint32_t count, uint64_t clear)
        {
            return count <= SMALL_ALWAYS || (count <= SMALL_TOKENS && clear >= count * SMALL_CLEAR_BYTES);
        }

        Plan planGradient(uint64_t rows, uint32_t dim, uint32_t count, bool small)
        {
            Plan     w{};
            uint64_t at   = 0;
            auto     take = [&](uint64_t bytes) {
                const uint64_t here = at;
                at += (bytes + 255u) / 256u * 256u;
                return here;
            };
            w.small    = small;
            const uint32_t tile = THREADS * (count < MANY_TOKENS ? FEW_ITEMS : MANY_ITEMS);
            w.tiles    = uint32_t((uint64_t(count) + tile - 1u) / tile);
            const uint32_t bits = log2Up(rows + 1u); // keys 0..rows
            w.passes    = (bits + SORT_BITS - 1u) / SORT_BITS;
            w.digitBits = (bits + w.passes - 1u) / w.passes;
            w.digitBits = w.digitBits < 8u ? 8u : w.digitBits;
            w.pairs[0] = take(uint64_t(count) * 8u);
            if(!w.small)
            {
                w.pairs[1] = take(uint64_t(count) * 8u);
                w.keys     = w.pairs[1]; // read by the first pass, which writes pairs[0]
                w.totals   = take(SORT_RADIX * 4u);
                w.counts   = take((uint64_t(w.tiles) << w.digitBits) * 4u);
            }
            // (pieces of the widest kind; narrower ones put fewer rows into a block, and fewer items)
            const uint32_t pieces = dim % 8u == 0u ? dim / 8u : dim % 4u == 0u ? dim / 4u : dim % 2u == 0u ? dim / 2u : dim;
            const uint32_t lanes  = rowLanesLog2(pieces);
            const uint32_t most   = SUM_ITEMS / (sumThreads(lanes) >> lanes); // that fit a block
            // Long chunks leave fewer pieces of runs behind, short ones make more threads: as many
            // as the device could hold of them.
            w.chunk = 8;
            while(w.chunk < 128u && w.chunk < most && uint64_t(count) * pieces > uint64_t(w.chunk) * DEVICE_THREADS)
                w.chunk *= 2u;
            // pieces of runs: two of each part, of which there are most where a row is cut into single
            // values and fewest of its pieces' threads fit a block
            const uint32_t single = rowLanesLog2(dim);
            const uint64_t parts  = partsOf(count, w.chunk, single);
            if(parts > 1u)
            {
                w.pieceKeys = take(parts * 8u);
                w.pieceSums = take(parts * 2u * dim * 4u);
            }
            w.bytes = at;
            return w;
        }

        struct GradientCall
        {
            Tokens      t;
            void const* grad;
            uint64_t    gradOuter, gradInner;
            void*       table;
            uint64_t    ldt;
            uint32_t    dim;
            float       scale;
            bool        accumulate;
            uint8_t*    workspace;
        };

#define B200WMMA_TRY(expr)       \
    do                           \
    {                            \
        const int rc__ = (expr); \
        if(rc__ != B200WMMA_OK)  \
            return rc__;         \
    } while(0)

        ClearParams clearParams(void* table, uint64_t ldt, uint32_t rows, uint32_t pieces)
        {
            return ClearParams{table, ldt, pieces, rowLanesLog2(pieces), 0, rows, 0};
        }

        // (row, token) of every token into the workspace, sorted; few tokens: rows without one
        // cleared on the way.
        template <typename OutT, int V, uint32_t BITS>
        int sortFewBits(GradientCall const& g, Plan const& w, cudaStream_t stream)
        {
            ClearParams c = clearParams(g.table, g.ldt, g.t.rows, g.dim / V);
            // a block to an SM, each with 16 KB of rows at least
            const uint64_t want = (uint64_t(g.t.rows) * g.dim * sizeof(OutT) + 16383u) / 16384u;
            c.blocks            = g.accumulate ? 0u : uint32_t(want < 147u ? want : 147u);
            static uint32_t done[64] = {};
            B200WMMA_TRY(optInSharedMemory(sortSmallKernel<OutT, V, BITS>, sizeof(SmallShared<BITS>), done));
            return cudaToStatus(launchOverlapped(sortSmallKernel<OutT, V, BITS>, dim3(1u + c.blocks), dim3(SMALL_THREADS),
                                                 sizeof(SmallShared<BITS>), stream, g.t, c, w.passes,
                                                 reinterpret_cast<uint2*>(g.workspace + w.pairs[0])));
        }

        template <typename OutT, int V>
        int sortFew(GradientCall const& g, Plan const& w, cudaStream_t stream)
        {
            return w.digitBits == 8u ? sortFewBits<OutT, V, 8>(g, w, stream)
                                     : w.digitBits == 9u ? sortFewBits<OutT, V, 9>(g, w, stream)
                                                         : sortFewBits<OutT, V, 10>(g, w, stream);
        }

        template <uint32_t ITEMS, uint32_t BITS>
        int sortMany(GradientCall const& g, Plan const& w, uint2** sorted, cudaStream_t stream)
        {
            auto       words = [&](uint64_t at) { return reinterpret_cast<uint32_t*>(g.workspace + at); };
            auto       pairs = [&](uint32_t i) { return reinterpret_cast<uint2*>(g.workspace + w.pairs[i]); };
            static uint32_t done[64] = {};
            B200WMMA_TRY(optInSharedMemory(scatterKernel<ITEMS, BITS>, sizeof(ScatterShared<ITEMS, BITS>), done));
            const dim3 grid(w.tiles);
            B200WMMA_TRY(cudaToStatus(launchOverlapped(keysKernel<ITEMS, BITS>, grid, dim3(THREADS), 0, stream, g.t,
                                                       words(w.keys), words(w.counts))));
            for(uint32_t pass = 0; pass < w.passes; ++pass)
            {
                uint2* from = pass ? pairs((pass - 1u) % 2u) : nullptr;
                if(pass > 0u)
                    B200WMMA_TRY(cudaToStatus(launchOverlapped(countKernel<ITEMS, BITS>, grid, dim3(THREADS), 0, stream, from,
                                                               g.t.count, pass, words(w.counts))));
                constexpr uint32_t radix = 1u << BITS;
                if(w.tiles > FEW_TILES)
                    B200WMMA_TRY(cudaToStatus(launchOverlapped(scanKernel, dim3((radix + SCAN_DIGITS - 1u) / SCAN_DIGITS),
                                                               dim3(SCAN_THREADS), 0, stream, words(w.counts), w.tiles, radix,
                                                               words(w.totals))));
                B200WMMA_TRY(cudaToStatus(launchOverlapped(scatterKernel<ITEMS, BITS>, grid, dim3(THREADS), sizeof(ScatterShared<ITEMS, BITS>),
                                                           stream, words(w.keys), from, g.t.count, pass,
                                                           w.tiles > FEW_TILES ? 0u : w.tiles,
                                                           words(w.counts), words(w.totals), pairs(pass % 2u))));
            }
            *sorted = pairs((w.passes - 1u) % 2u);
            return B200WMMA_OK;
        }

        template <uint32_t ITEMS>
        int sortDigits(GradientCall const& g, Plan const& w, uint2** sorted, cudaStream_t stream)
        {
            return w.digitBits == 8u ? sortMany<ITEMS, 8>(g, w, sorted, stream)
                                     : w.digitBits == 9u ? sortMany<ITEMS, 9>(g, w, sorted, stream)
                                                         : sortMany<ITEMS, 10>(g, w, sorted, stream);
        }

        // The sums of chunks, with pieces of `V` values, and rows cleared beside them where the
        // sort has not done that.
        template <typename T, typename OutT, int V>
        int sumChunks(GradientCall const& g, Plan const& w, SumParams p, cudaStream_t stream)
        {
            p.pieces    = g.dim / V;
            p.lanesLog2 = rowLanesLog2(p.pieces);
            p.slices    = (p.pieces + (1u << p.lanesLog2) - 1u) >> p.lanesLog2;
            const uint32_t threads = sumThreads(p.lanesLog2);
            const uint64_t blocks  = uint64_t(p.parts) * p.slices;
            // rows may lie on wider boundaries than those of the gradient: clear by the narrower
            ClearParams c = clearParams(g.table, g.ldt, g.t.rows, p.pieces);
            c.lanesLog2   = c.lanesLog2 < log2Up(threads) ? c.lanesLog2 : log2Up(threads);
            if(!w.small && !g.accumulate)
            {
                const uint64_t rowBytes = uint64_t(g.dim) * sizeof(OutT);
                c.rowsPerBlock          = rowBytes >= 65536u ? 1u : uint32_t(65536u / rowBytes);
                c.rowsPerBlock          = c.rowsPerBlock > SUM_ITEMS ? SUM_ITEMS : c.rowsPerBlock;
                c.blocks                = (g.t.rows + c.rowsPerBlock - 1u) / c.rowsPerBlock;
            }
            if(blocks + c.blocks > 0x7fffffffull)
                return B200WMMA_ERR_TOO_LARGE;
            p.blocks = uint32_t(blocks);
            return cudaToStatus(launchOverlapped(sumKernel<T, OutT, V>, dim3(p.blocks + c.blocks), dim3(threads),
                                                 threads * Ring<T, V>::DEPTH * Ring<T, V>::BYTES, stream, p, c));
        }

        template <typename OutT, int V>
        int joinPieces(GradientCall const& g, SumParams p, cudaStream_t stream)
        {
            p.pieces    = g.dim / V;
            // at most a warp to a row, so that a block has eight groups for the long runs (16384
            // tokens of 4096, where the most frequent one has 75 pieces: 18 us with 256 threads to a
            // row, 6 with 32)
            p.lanesLog2 = rowLanesLog2(p.pieces) < 5u ? rowLanesLog2(p.pieces) : 5u;
            p.slices    = (p.pieces + (1u << p.lanesLog2) - 1u) >> p.lanesLog2;
            const uint32_t groups = THREADS >> p.lanesLog2;
            const uint64_t blocks = (uint64_t(p.parts) + groups - 1u) / groups * p.slices;
            if(blocks > 0x7fffffffull)
                return B200WMMA_ERR_TOO_LARGE;
            return cudaToStatus(launchOverlapped(joinKernel<OutT, V>, dim3(uint32_t(blocks)), dim3(THREADS), 0, stream, p));
        }

        template <typename T, typename OutT>
        int gradient(GradientCall const& g, cudaStream_t stream)
        {
            const uint64_t clear = g.accumulate ? 0u : uint64_t(g.t.rows) * g.dim * sizeof(OutT);
            const Plan     w  = planGradient(g.t.rows, g.dim, g.t.count, sortsSmall(g.t.count, clear));
            const uint32_t vt = pieceSize(g.dim, g.table, sizeof(OutT), 8, g.ldt);
            // (the gradient comes in copies of 16 bytes at most; two for a piece of 32 would each touch half of
            // a sector: 236000 rows of 208 f32 take 80 us with eight values to a piece, 61 with four)
            const uint32_t most = sizeof(T) == 4 && vt == 8u ? 4u : vt;
            const uint32_t vg   = pieceSize(g.dim, g.grad, sizeof(T), most, g.gradOuter, g.gradInner);
            uint2*         sorted = reinterpret_cast<uint2*>(g.workspace + w.pairs[0]);
            if(w.small)
                B200WMMA_TRY(withPiece(vt, [&](auto V) { return sortFew<OutT, V.value>(g, w, stream); }));
            else
                B200WMMA_TRY(g.t.count < MANY_TOKENS ? sortDigits<FEW_ITEMS>(g, w, &sorted, stream)
                                                     : sortDigits<MANY_ITEMS>(g, w, &sorted, stream));
            SumParams p{};
            p.sorted     = sorted;
            p.grad       = g.grad;
            p.gradOuter  = g.gradOuter;
            p.gradInner  = g.gradInner;
            p.inner      = g.t.inner;
            p.n          = g.t.count;
            p.chunk      = w.chunk;
            p.parts      = uint32_t(partsOf(g.t.count, w.chunk, rowLanesLog2(g.dim / vg)));
            p.rows       = g.t.rows;
            p.table      = g.table;
            p.ldt        = g.ldt;
            p.scale      = g.scale;
            p.accumulate = g.accumulate ? 1u : 0u;
            if(p.parts > 1u)
            {
                p.pieceKeys = reinterpret_cast<uint32_t*>(g.workspace + w.pieceKeys);
                p.pieceSums = reinterpret_cast<float*>(g.workspace + w.pieceSums);
            }
            B200WMMA_TRY(withPiece(vg, [&](auto V) {
                if constexpr(sizeof(T) * V.value > 16)
                    return int(B200WMMA_ERR_INVALID_ARG); // never
                else
                    return sumChunks<T, OutT, V.value>(g, w, p, stream);
            }));
            if(p.parts > 1u)
                B200WMMA_TRY(withPiece(vt, [&](auto V) { return joinPieces<OutT, V.value>(g, p, stream); }));
            return B200WMMA_OK;
        }
#undef B200WMMA_TRY

        template <typename T>
        int gradientFrom(int out, GradientCall const& g, cudaStream_t stream)
        {
            switch(out)
            {
            case B200WMMA_F16:
                return gradient<T, __half>(g, stream);
            case B200WMMA_BF16:
                return gradient<T, __nv_bfloat16>(g, stream);
            }
            return gradient<T, float>(g, stream);
        }

        // Sizes and ids, which both directions check alike.
        int checkTokens(uint64_t rows, uint32_t dim, uint64_t outer, uint32_t inner, void const* table,
                        uint64_t ldt, void const* ids, int idBytes, int64_t const* first, void const* values,
                        int tableType, int valuesType)
        {
            if(!table || !ids || !values || rows == 0 || dim == 0 || outer == 0 || inner == 0 || ldt < dim
               || (idBytes != 4 && idBytes != 8))
                return B200WMMA_ERR_INVALID_ARG;
            if(!valueType(tableType) || !valueType(valuesType))
                return B200WMMA_ERR_UNSUPPORTED;
            if(!aligned(table, dtypeSize(tableType)) || !aligned(values, dtypeSize(valuesType))
               || !aligned(ids, uint64_t(idBytes)) || !aligned(first, 8))
                return B200WMMA_ERR_ALIGNMENT;
            // rows and tokens are counted in 31 bits
            if(rows >= NO_ROW || outer > 0x7ffff000ull / inner || dim > 0x100000u)
                return B200WMMA_ERR_TOO_LARGE;
            return B200WMMA_OK;
        }
    } // namespace
} // namespace b200wmma

using namespace b200wmma;

extern "C" {

int b200wmma_embedding(int table_dtype, int out_dtype, uint64_t rows, uint32_t dim, uint64_t outer,
                       uint32_t inner, const void* table, uint64_t ldt, const void* ids, int id_bytes,
                       uint64_t ids_outer, uint64_t ids_inner, const int64_t* first, void* out,
                       uint64_t out_outer, uint64_t out_inner, double scale, void* stream)
{
    const int rc = checkTokens(rows, dim, outer, inner, table, ldt, ids, id_bytes, first, out,
                               table_dtype, out_dtype);
    if(rc != B200WMMA_OK)
        return rc;
    if(rowsOverlap(outer, out_outer, inner, out_inner, dim)) // which row would remain is nobody's choice
        return B200WMMA_ERR_INVALID_ARG;
    LookupParams p{};
    p.t = Tokens{ids, first, ids_outer, ids_inner, uint32_t(outer * inner), uint32_t(rows), Divisor(inner), id_bytes == 8 ? 1u : 0u};
    p.table    = table;
    p.out      = out;
    p.ldt      = ldt;
    p.outOuter = out_outer;
    p.outInner = out_inner;
    p.scale    = float(scale);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch(table_dtype)
    {
    case B200WMMA_F16:
        return lookupFrom<__half>(out_dtype, p, dim, s);
    case B200WMMA_BF16:
        return lookupFrom<__nv_bfloat16>(out_dtype, p, dim, s);
    }
    return lookupFrom<float>(out_dtype, p, dim, s);
}

uint64_t b200wmma_embedding_grad_workspace(uint64_t rows, uint32_t dim, uint64_t outer, uint32_t inner)
{
    if(rows == 0 || dim == 0 || outer == 0 || inner == 0 || rows >= NO_ROW || outer > 0x7ffff000ull / inner)
        return 0;
    // (whichever way the call takes: that of many tokens needs more)
    const uint32_t count = uint32_t(outer * inner);
    return planGradient(rows, dim, count, sortsSmall(count, 0)).bytes;
}

int b200wmma_embedding_grad(int grad_dtype, int table_dtype, uint64_t rows, uint32_t dim, uint64_t outer,
                            uint32_t inner, const void* grad, uint64_t grad_outer, uint64_t grad_inner,
                            const void* ids, int id_bytes, uint64_t ids_outer, uint64_t ids_inner,
                            const int64_t* first, void* table_grad, uint64_t ldt, double scale,
                            int accumulate, void* workspace, uint64_t workspace_bytes, void* stream)
{
    const int rc = checkTokens(rows, dim, outer, inner, table_grad, ldt, ids, id_bytes, first, grad,
                               table_dtype, grad_dtype);
    if(rc != B200WMMA_OK)
        return rc;
    if(!workspace || workspace_bytes < b200wmma_embedding_grad_workspace(rows, dim, outer, inner))
        return B200WMMA_ERR_INVALID_ARG;
    if(!aligned(workspace, 256))
        return B200WMMA_ERR_ALIGNMENT;
    const GradientCall g{Tokens{ids, first, ids_outer, ids_inner, uint32_t(outer * inner), uint32_t(rows), Divisor(inner), id_bytes == 8 ? 1u : 0u},
                         grad, grad_outer, grad_inner, table_grad, ldt, dim, float(scale), accumulate != 0,
                         static_cast<uint8_t*>(workspace)};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch(grad_dtype)
    {
    case B200WMMA_F16:
        return gradientFrom<__half>(table_dtype, g, s);
    case B200WMMA_BF16:
        return gradientFrom<__nv_bfloat16>(table_dtype, g, s);
    }
    return gradientFrom<float>(table_dtype, g, s);
}
}
