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
// result depends on its arguments alone: tokens are sorted by row (a stable radix sort), then
// every run of equal rows is summed in token order, in fp32, by cutting the sorted tokens into
// chunks; a run inside one chunk is written at once, the pieces of a run that crosses chunks go
// to the workspace, which the next, much smaller level treats as its tokens.
#include "common.cuh"
#include "mx_format.cuh"
#include "rocwmma/rocwmma_block.hpp"

namespace b200wmma
{
    using rocwmma::block::grid_dependency_wait;
    using rocwmma::block::grid_launch_dependents;

    namespace
    {
        constexpr uint32_t THREADS = 256;
        constexpr uint32_t NO_ROW  = 0x7fffffffu; // no token, or no row of the table
        constexpr uint32_t EMPTY   = 0x80000000u; // part of a run, but adds nothing to it

        // The tokens of a call.
        struct Tokens
        {
            void const*    ids;
            int64_t const* first;
            uint64_t       idsOuter, idsInner; // strides, elements
            uint32_t       count, inner, rows;
            uint32_t       wide; // 64-bit ids
        };

        __device__ inline uint32_t rowOf(Tokens const& t, uint32_t token, uint32_t& outer, uint32_t& inner)
        {
            outer = token;
            inner = 0;
            if(t.inner > 1u)
            {
                outer = token / t.inner;
                inner = token - outer * t.inner;
            }
            const uint64_t at = uint64_t(outer) * t.idsOuter + uint64_t(inner) * t.idsInner;
            const int64_t  id = t.wide ? static_cast<int64_t const*>(t.ids)[at]
                                       : int64_t(static_cast<int32_t const*>(t.ids)[at]);
            int64_t row = id, end = t.rows;
            if(t.first)
            {
                const int64_t begin = t.first[inner];
                end                 = t.first[inner + 1];
                row                 = begin + id;
                if(begin < 0 || end > int64_t(t.rows) || id < 0 || id >= end - begin)
                    return NO_ROW;
            }
            return row >= 0 && row < end ? uint32_t(row) : NO_ROW;
        }

        // V values of a row: 16 or 32 bytes with V = 8, one element with V = 1.
        template <typename T, int V>
        struct Piece
        {
            static constexpr int BYTES = int(sizeof(T)) * V;
            T                    v[V];
        };
        template <typename T, int V>
        __device__ inline void loadPiece(T const* p, float (&f)[V])
        {
            if constexpr(V == 1)
                f[0] = toFloat(*p);
            else
            {
                constexpr int N = int(sizeof(T)) * V / 16;
                uint4         raw[N];
#pragma unroll
                for(int i = 0; i < N; ++i)
                    raw[i] = reinterpret_cast<uint4 const*>(p)[i];
#pragma unroll
                for(int i = 0; i < V; ++i)
                    f[i] = toFloat(reinterpret_cast<T const*>(raw)[i]);
            }
        }
        template <typename T, int V>
        __device__ inline void storePiece(T* p, float const (&f)[V])
        {
            if constexpr(V == 1)
                *p = fromFloat<T>(f[0]);
            else
            {
                constexpr int N = int(sizeof(T)) * V / 16;
                alignas(16) T v[V];
#pragma unroll
                for(int i = 0; i < V; ++i)
                    v[i] = fromFloat<T>(f[i]);
#pragma unroll
                for(int i = 0; i < N; ++i)
                    __stcs(reinterpret_cast<uint4*>(p) + i, reinterpret_cast<uint4 const*>(v)[i]);
            }
        }

        // ---- lookup ----------------------------------------------------------------------
        struct LookupParams
        {
            Tokens      t;
            void const* table;
            void*       out;
            uint64_t    ldt, outOuter, outInner;
            uint32_t    pieces, lanesLog2; // pieces of a row; threads side by side on a row
            float       scale;
        };

        // A thread moves one piece of U tokens; 2^lanesLog2 neighbours share the tokens.
        template <typename T, typename OutT, int V, int U>
        __global__ void __launch_bounds__(THREADS) lookupKernel(const LookupParams p)
        {
            const uint32_t lanes = 1u << p.lanesLog2;
            const uint32_t piece = blockIdx.y * lanes + (threadIdx.x & (lanes - 1u));
            const uint32_t perStep = THREADS >> p.lanesLog2;
            const uint32_t token0  = blockIdx.x * (perStep * U) + (threadIdx.x >> p.lanesLog2);
            grid_dependency_wait();
            grid_launch_dependents();
            if(piece >= p.pieces)
                return;
            float    v[U][V];
            uint64_t at[U];
            bool     in[U];
#pragma unroll
            for(int u = 0; u < U; ++u)
            {
                const uint32_t token = token0 + u * perStep;
                in[u]                = token < p.t.count;
                uint32_t outer = 0, inner = 0;
                const uint32_t row = in[u] ? rowOf(p.t, token, outer, inner) : NO_ROW;
                at[u] = uint64_t(outer) * p.outOuter + uint64_t(inner) * p.outInner + uint64_t(piece) * V;
                if(row != NO_ROW)
                    loadPiece<T, V>(static_cast<T const*>(p.table) + uint64_t(row) * p.ldt + uint64_t(piece) * V, v[u]);
                else
                {
#pragma unroll
                    for(int i = 0; i < V; ++i)
                        v[u][i] = 0.0f;
                }
                // an unwritten row stays a zero: scale may be infinite or NaN
                if(row != NO_ROW)
                {
#pragma unroll
                    for(int i = 0; i < V; ++i)
                        v[u][i] *= p.scale;
                }
            }
#pragma unroll
            for(int u = 0; u < U; ++u)
                if(in[u])
                    storePiece<OutT, V>(static_cast<OutT*>(p.out) + at[u], v[u]);
        }

        // ---- sorting tokens by row ---------------------------------------------------------
        constexpr uint32_t SORT_ITEMS  = 16; // keys of a thread
        constexpr uint32_t SORT_TILE   = THREADS * SORT_ITEMS;
        constexpr uint32_t RADIX       = 256;
        constexpr uint32_t SORT_WARPS  = THREADS / 32;

        // Row of every token, and a bit for every row that has one.
        __global__ void __launch_bounds__(THREADS) keysKernel(const Tokens t, uint32_t* keys, uint32_t* touched)
        {
            grid_dependency_wait();
            grid_launch_dependents();
            const uint32_t token = blockIdx.x * THREADS + threadIdx.x;
            if(token >= t.count)
                return;
            uint32_t       outer, inner;
            const uint32_t row = rowOf(t, token, outer, inner);
            keys[token]        = row == NO_ROW ? t.rows : row; // behind every row
            if(row != NO_ROW && touched)
                atomicOr(&touched[row / 32u], 1u << (row % 32u));
        }

        // counts[digit][tile]
        __global__ void __launch_bounds__(THREADS)
            countKernel(uint32_t const* keys, uint32_t n, uint32_t shift, uint32_t tiles, uint32_t* counts)
        {
            __shared__ uint32_t bins[RADIX];
            grid_dependency_wait();
            grid_launch_dependents();
            bins[threadIdx.x] = 0;
            __syncthreads();
#pragma unroll
            for(uint32_t i = 0; i < SORT_ITEMS; ++i)
            {
                const uint64_t at = uint64_t(blockIdx.x) * SORT_TILE + i * THREADS + threadIdx.x;
                if(at < n)
                    atomicAdd(&bins[(keys[at] >> shift) % RADIX], 1u);
            }
            __syncthreads();
            counts[threadIdx.x * tiles + blockIdx.x] = bins[threadIdx.x];
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

        // One block per digit: its row of counts becomes its exclusive sums, the total goes to
        // totals[digit].
        __global__ void __launch_bounds__(THREADS) scanKernel(uint32_t* counts, uint32_t tiles, uint32_t* totals)
        {
            __shared__ uint32_t warps[SORT_WARPS];
            grid_dependency_wait();
            grid_launch_dependents();
            uint32_t* row = counts + uint64_t(blockIdx.x) * tiles;
            uint32_t  sum = 0;
            for(uint32_t t0 = 0; t0 < tiles; t0 += THREADS)
            {
                const uint32_t t = t0 + threadIdx.x;
                uint32_t       total;
                const uint32_t before = blockScan(t < tiles ? row[t] : 0u, warps, total);
                if(t < tiles)
                    row[t] = sum + before;
                sum += total;
            }
            if(threadIdx.x == 0)
                totals[blockIdx.x] = sum;
        }

        // Moves every key of a tile, with its token, to its place among the keys of this digit:
        // those of smaller digits, of earlier tiles, of earlier warps, of earlier rows of 32 and
        // of smaller lanes come first.  tokensIn == nullptr: key i belongs to token i.
        __global__ void __launch_bounds__(THREADS)
            scatterKernel(uint32_t const* keysIn, uint32_t const* tokensIn, uint32_t n, uint32_t shift,
                          uint32_t tiles, uint32_t const* counts, uint32_t const* totals,
                          uint32_t* keysOut, uint32_t* tokensOut)
        {
            __shared__ uint32_t bins[SORT_WARPS][RADIX];
            __shared__ uint32_t warps[SORT_WARPS];
            const uint32_t      warp = threadIdx.x / 32u, lane = threadIdx.x % 32u;
            grid_dependency_wait();
            grid_launch_dependents();
#pragma unroll
            for(uint32_t w = 0; w < SORT_WARPS; ++w)
                bins[w][threadIdx.x] = 0;
            __syncthreads();
            const uint64_t first = uint64_t(blockIdx.x) * SORT_TILE + warp * (32u * SORT_ITEMS) + lane;
            uint32_t       key[SORT_ITEMS], rank[SORT_ITEMS];
#pragma unroll
            for(uint32_t i = 0; i < SORT_ITEMS; ++i)
            {
                const uint64_t at = first + i * 32u;
                key[i]            = at < n ? keysIn[at] : 0xffffffffu;
            }
#pragma unroll
            for(uint32_t i = 0; i < SORT_ITEMS; ++i)
            {
                const bool     in    = first + i * 32u < n;
                const uint32_t digit = (key[i] >> shift) % RADIX;
                const uint32_t peers = __match_any_sync(0xffffffffu, in ? digit : RADIX);
                const uint32_t before = in ? bins[warp][digit] : 0u;
                rank[i]               = before + __popc(peers & ((1u << lane) - 1u));
                __syncwarp();
                if(in && (peers >> lane) == 1u) // the last of its digit
                    bins[warp][digit] = rank[i] + 1u;
                __syncwarp();
            }
            __syncthreads();
            // thread = digit: where the keys of each warp go
            {
                uint32_t       total;
                const uint32_t base = blockScan(totals[threadIdx.x], warps, total)
                                      + counts[threadIdx.x * tiles + blockIdx.x];
                uint32_t sum = base;
#pragma unroll
                for(uint32_t w = 0; w < SORT_WARPS; ++w)
                {
                    const uint32_t count = bins[w][threadIdx.x];
                    bins[w][threadIdx.x] = sum;
                    sum += count;
                }
            }
            __syncthreads();
#pragma unroll
            for(uint32_t i = 0; i < SORT_ITEMS; ++i)
            {
                const uint64_t at = first + i * 32u;
                if(at < n)
                {
                    const uint32_t to = bins[warp][(key[i] >> shift) % RADIX] + rank[i];
                    keysOut[to]       = key[i];
                    tokensOut[to]     = tokensIn ? tokensIn[at] : uint32_t(at);
                }
            }
        }

        // ---- summing runs ------------------------------------------------------------------
        struct SumParams
        {
            uint32_t const* keys; // of the items, equal rows next to each other
            uint32_t const* tokens; // nullptr: item i is row i of `grad`
            void const*     grad;
            uint64_t        gradOuter, gradInner;
            uint32_t        inner;
            uint32_t        n, chunk, rows;
            uint32_t        pieces, lanesLog2;
            void*           table;
            uint64_t        ldt;
            float           scale;
            uint32_t        accumulate;
            uint32_t*       pieceKeys; // two of each chunk: run from the left, run to the right
            float*          pieceSums; // rows of `pieces * V`
        };

        template <typename T, typename OutT, int V>
        __global__ void __launch_bounds__(THREADS) sumKernel(const SumParams p)
        {
            constexpr uint32_t U     = 8;
            const uint32_t     lanes = 1u << p.lanesLog2;
            const uint32_t piece = blockIdx.y * lanes + (threadIdx.x & (lanes - 1u));
            const uint64_t chunkIdx = uint64_t(blockIdx.x) * (THREADS >> p.lanesLog2) + (threadIdx.x >> p.lanesLog2);
            const uint64_t begin = chunkIdx * p.chunk;
            grid_dependency_wait();
            grid_launch_dependents();
            if(piece >= p.pieces || begin >= p.n)
                return;
            const uint32_t end = uint32_t(min(uint64_t(p.n), begin + p.chunk));
            const uint64_t width = uint64_t(p.pieces) * V;
            const bool     marks = piece == 0u && p.pieceKeys != nullptr;
            const uint32_t before = begin > 0 ? p.keys[begin - 1] & ~EMPTY : NO_ROW;
            const uint32_t after  = end < p.n ? p.keys[end] & ~EMPTY : NO_ROW;

            float    sum[V];
            uint32_t run = NO_ROW; // row of the current run
            bool     fromLeft = false, left = false, right = false;
            uint32_t leftKey = NO_ROW, rightKey = NO_ROW;
            auto flush = [&](bool last) {
                if(run >= p.rows)
                    return;
                const bool toRight = last && after == run;
                if(!fromLeft && !toRight)
                {
                    OutT* at = static_cast<OutT*>(p.table) + uint64_t(run) * p.ldt + uint64_t(piece) * V;
                    float v[V];
                    if(p.accumulate)
                    {
                        loadPiece<OutT, V>(at, v);
#pragma unroll
                        for(int i = 0; i < V; ++i)
                            v[i] = fmaf(sum[i], p.scale, v[i]);
                    }
                    else
                    {
#pragma unroll
                        for(int i = 0; i < V; ++i)
                            v[i] = sum[i] * p.scale;
                    }
                    storePiece<OutT, V>(at, v);
                    return;
                }
                float* at = p.pieceSums + (2u * chunkIdx + (fromLeft ? 0u : 1u)) * width + uint64_t(piece) * V;
#pragma unroll
                for(int i = 0; i < V; ++i)
                    at[i] = sum[i];
                if(fromLeft)
                {
                    left    = true;
                    leftKey = run;
                    if(toRight) // the run goes on: keep it one across this chunk's second place
                        rightKey = run | EMPTY;
                }
                else
                {
                    right    = true;
                    rightKey = run;
                }
            };

            for(uint32_t i0 = uint32_t(begin); i0 < end; i0 += U)
            {
                float    v[U][V];
                uint32_t key[U];
#pragma unroll
                for(uint32_t u = 0; u < U; ++u)
                {
                    const uint32_t i = i0 + u;
                    key[u]           = i < end ? p.keys[i] : NO_ROW | EMPTY;
                    if((key[u] & EMPTY) == 0u && key[u] < p.rows)
                    {
                        const uint32_t token = p.tokens ? p.tokens[i] : i;
                        uint64_t       at;
                        if(p.inner > 1u)
                        {
                            const uint32_t outer = token / p.inner;
                            at = uint64_t(outer) * p.gradOuter + uint64_t(token - outer * p.inner) * p.gradInner;
                        }
                        else
                            at = uint64_t(token) * p.gradOuter;
                        loadPiece<T, V>(static_cast<T const*>(p.grad) + at + uint64_t(piece) * V, v[u]);
                    }
                    else
                    {
#pragma unroll
                        for(int j = 0; j < V; ++j)
                            v[u][j] = 0.0f;
                    }
                }
#pragma unroll
                for(uint32_t u = 0; u < U; ++u)
                {
                    if(i0 + u >= end)
                        break;
                    const uint32_t row = key[u] & ~EMPTY;
                    if(row != run)
                    {
                        flush(false);
                        run      = row;
                        fromLeft = i0 + u == begin && before == row;
#pragma unroll
                        for(int j = 0; j < V; ++j)
                            sum[j] = v[u][j];
                    }
                    else if((key[u] & EMPTY) == 0u)
                    {
#pragma unroll
                        for(int j = 0; j < V; ++j)
                            sum[j] += v[u][j];
                    }
                }
            }
            flush(true);
            if(marks)
            {
                p.pieceKeys[2u * chunkIdx]      = leftKey;
                p.pieceKeys[2u * chunkIdx + 1u] = rightKey;
            }
        }

        // Rows without a token.
        template <typename OutT, int V>
        __global__ void __launch_bounds__(THREADS)
            clearKernel(OutT* table, uint64_t ldt, uint32_t rows, uint32_t pieces, uint32_t lanesLog2,
                        uint32_t const* touched)
        {
            const uint32_t lanes = 1u << lanesLog2;
            const uint64_t row   = uint64_t(blockIdx.x) * (THREADS >> lanesLog2) + (threadIdx.x >> lanesLog2);
            grid_dependency_wait();
            grid_launch_dependents();
            if(row >= rows || (touched[row / 32u] >> (row % 32u)) & 1u)
                return;
            float zero[V];
#pragma unroll
            for(int i = 0; i < V; ++i)
                zero[i] = 0.0f;
            for(uint32_t piece = threadIdx.x & (lanes - 1u); piece < pieces; piece += lanes)
                storePiece<OutT, V>(table + row * ldt + uint64_t(piece) * V, zero);
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
        // Threads side by side on a row of `pieces`: enough, but no more than a block has.
        uint32_t lanesFor(uint32_t pieces)
        {
            const uint32_t l = log2Up(pieces);
            return l > 8u ? 8u : l;
        }

        template <typename T, typename OutT, int V>
        int lookup(LookupParams p, cudaStream_t stream)
        {
            const uint32_t perStep = THREADS >> p.lanesLog2;
            const uint32_t lanes   = 1u << p.lanesLog2;
            const uint32_t across  = (p.pieces + lanes - 1u) / lanes;
            // four tokens a thread once that still fills the device
            const bool     many   = uint64_t(p.t.count) * across / perStep >= 4u * 148u * 8u;
            const uint32_t each   = perStep * (many ? 4u : 1u);
            const dim3     grid((p.t.count + each - 1u) / each, across);
            return cudaToStatus(many ? launchOverlapped(lookupKernel<T, OutT, V, 4>, grid, dim3(THREADS), 0, stream, p)
                                     : launchOverlapped(lookupKernel<T, OutT, V, 1>, grid, dim3(THREADS), 0, stream, p));
        }

        template <typename T, typename OutT>
        int lookupTyped(LookupParams p, uint32_t dim, cudaStream_t stream)
        {
            // pieces of eight values where every row of the table and of the output starts on a
            // 16-byte boundary, single values elsewhere
            const bool wide = dim % 8u == 0u && aligned(p.table, 16) && aligned(p.out, 16)
                              && p.ldt * sizeof(T) % 16 == 0 && p.outOuter * sizeof(OutT) % 16 == 0
                              && p.outInner * sizeof(OutT) % 16 == 0;
            p.pieces    = wide ? dim / 8u : dim;
            p.lanesLog2 = lanesFor(p.pieces);
            return wide ? lookup<T, OutT, 8>(p, stream) : lookup<T, OutT, 1>(p, stream);
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

        // The workspace of the gradient; offsets in bytes.
        constexpr uint32_t MAX_LEVELS = 8;
        struct Plan
        {
            uint64_t keys[2], tokens[2], counts, totals, touched, bytes;
            uint64_t touchedBytes;
            uint32_t tiles, passes, levels;
            uint32_t n[MAX_LEVELS], chunk[MAX_LEVELS];
            uint64_t pieceKeys[MAX_LEVELS], pieceSums[MAX_LEVELS];
        };

        Plan planGradient(uint64_t rows, uint32_t dim, uint32_t count)
        {
            Plan     w{};
            uint64_t at   = 0;
            auto     take = [&](uint64_t bytes) {
                const uint64_t here = at;
                at += (bytes + 255u) / 256u * 256u;
                return here;
            };
            w.tiles  = uint32_t((uint64_t(count) + SORT_TILE - 1) / SORT_TILE);
            w.passes = (log2Up(rows + 1u) + 7u) / 8u; // keys 0..rows
            if(w.passes == 0)
                w.passes = 1;
            w.touchedBytes = (rows + 31u) / 32u * 4u;
            w.touched      = take(w.touchedBytes);
            w.totals       = take(RADIX * 4u);
            w.counts       = take(uint64_t(w.tiles) * RADIX * 4u);
            for(int i = 0; i < 2; ++i)
            {
                w.keys[i]   = take(uint64_t(count) * 4u);
                w.tokens[i] = take(uint64_t(count) * 4u);
            }
            uint32_t n = count;
            while(true)
            {
                const uint32_t level = w.levels++;
                w.n[level]           = n;
                w.chunk[level]       = level == 0 ? 32u : 128u;
                const uint32_t chunks = (n + w.chunk[level] - 1u) / w.chunk[level];
                if(chunks <= 1u)
                    break;
                n                    = 2u * chunks;
                w.pieceKeys[level]   = take(uint64_t(n) * 4u);
                w.pieceSums[level]   = take(uint64_t(n) * dim * 4u);
            }
            w.bytes = at;
            return w;
        }

        template <typename T, typename OutT, int V>
        int sumLevel(SumParams p, uint32_t dim, cudaStream_t stream)
        {
            p.pieces    = dim / V;
            p.lanesLog2 = lanesFor(p.pieces);
            if(p.lanesLog2 > 5u)
                p.lanesLog2 = 5u; // one chunk to a warp at most
            const uint32_t lanes  = 1u << p.lanesLog2;
            const uint32_t chunks = uint32_t((uint64_t(p.n) + p.chunk - 1u) / p.chunk);
            const uint32_t per    = THREADS >> p.lanesLog2;
            const dim3     grid((chunks + per - 1u) / per, (p.pieces + lanes - 1u) / lanes);
            return cudaToStatus(launchOverlapped(sumKernel<T, OutT, V>, grid, dim3(THREADS), 0, stream, p));
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

        template <typename T, typename OutT>
        int gradient(GradientCall const& g, cudaStream_t stream)
        {
            const Plan w     = planGradient(g.t.rows, g.dim, g.t.count);
            auto       words = [&](uint64_t at) { return reinterpret_cast<uint32_t*>(g.workspace + at); };
            uint32_t*  touched = g.accumulate ? nullptr : words(w.touched);
            const bool wideTable = g.dim % 8u == 0u && aligned(g.table, 16) && g.ldt * sizeof(OutT) % 16 == 0;
            const bool wide = wideTable && aligned(g.grad, 16) && g.gradOuter * sizeof(T) % 16 == 0
                              && g.gradInner * sizeof(T) % 16 == 0;
#define B200WMMA_TRY(expr)          \
    do                              \
    {                               \
        const int rc__ = (expr);    \
        if(rc__ != B200WMMA_OK)     \
            return rc__;            \
    } while(0)
            if(touched)
                B200WMMA_CUDA_TRY(cudaMemsetAsync(touched, 0, w.touchedBytes, stream));
            B200WMMA_TRY(cudaToStatus(launchOverlapped(keysKernel, dim3((g.t.count + THREADS - 1u) / THREADS),
                                                       dim3(THREADS), 0, stream, g.t, words(w.keys[0]), touched)));
            for(uint32_t pass = 0; pass < w.passes; ++pass)
            {
                const uint32_t from = pass % 2u, to = 1u - from, shift = 8u * pass;
                B200WMMA_TRY(cudaToStatus(launchOverlapped(countKernel, dim3(w.tiles), dim3(THREADS), 0, stream,
                                                           words(w.keys[from]), g.t.count, shift, w.tiles, words(w.counts))));
                B200WMMA_TRY(cudaToStatus(launchOverlapped(scanKernel, dim3(RADIX), dim3(THREADS), 0, stream,
                                                           words(w.counts), w.tiles, words(w.totals))));
                B200WMMA_TRY(cudaToStatus(launchOverlapped(scatterKernel, dim3(w.tiles), dim3(THREADS), 0, stream,
                                                           words(w.keys[from]), pass ? words(w.tokens[from]) : nullptr,
                                                           g.t.count, shift, w.tiles, words(w.counts), words(w.totals),
                                                           words(w.keys[to]), words(w.tokens[to]))));
            }
            if(touched)
            {
                const uint32_t pieces = wideTable ? g.dim / 8u : g.dim, lanes = lanesFor(pieces);
                const uint32_t blocks = uint32_t((uint64_t(g.t.rows) + (THREADS >> lanes) - 1u) / (THREADS >> lanes));
                B200WMMA_TRY(cudaToStatus(wideTable
                    ? launchOverlapped(clearKernel<OutT, 8>, dim3(blocks), dim3(THREADS), 0, stream,
                                       static_cast<OutT*>(g.table), g.ldt, g.t.rows, pieces, lanes, touched)
                    : launchOverlapped(clearKernel<OutT, 1>, dim3(blocks), dim3(THREADS), 0, stream,
                                       static_cast<OutT*>(g.table), g.ldt, g.t.rows, pieces, lanes, touched)));
            }
            for(uint32_t level = 0; level < w.levels; ++level)
            {
                const bool more = level + 1u < w.levels;
                SumParams  p{};
                p.n     = w.n[level];
                p.chunk = w.chunk[level];
                p.rows  = g.t.rows;
                p.table = g.table;
                p.ldt   = g.ldt;
                p.scale = g.scale;
                p.accumulate = g.accumulate ? 1u : 0u;
                p.pieceKeys  = more ? words(w.pieceKeys[level]) : nullptr;
                p.pieceSums  = more ? reinterpret_cast<float*>(g.workspace + w.pieceSums[level]) : nullptr;
                if(level == 0)
                {
                    p.keys      = words(w.keys[w.passes % 2u]);
                    p.tokens    = words(w.tokens[w.passes % 2u]);
                    p.grad      = g.grad;
                    p.gradOuter = g.gradOuter;
                    p.gradInner = g.gradInner;
                    p.inner     = g.t.inner;
                    B200WMMA_TRY(wide ? (sumLevel<T, OutT, 8>(p, g.dim, stream)) : (sumLevel<T, OutT, 1>(p, g.dim, stream)));
                }
                else
                {
                    p.keys      = words(w.pieceKeys[level - 1u]);
                    p.grad      = g.workspace + w.pieceSums[level - 1u];
                    p.gradOuter = g.dim;
                    p.inner     = 1;
                    B200WMMA_TRY(wideTable ? (sumLevel<float, OutT, 8>(p, g.dim, stream))
                                           : (sumLevel<float, OutT, 1>(p, g.dim, stream)));
                }
            }
#undef B200WMMA_TRY
            return B200WMMA_OK;
        }

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
            // rows and tokens are counted in 31 bits; a grid's second dimension has 16
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
    LookupParams p{};
    p.t = Tokens{ids, first, ids_outer, ids_inner, uint32_t(outer * inner), inner, uint32_t(rows), id_bytes == 8 ? 1u : 0u};
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
    return planGradient(rows, dim, uint32_t(outer * inner)).bytes;
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
    const GradientCall g{Tokens{ids, first, ids_outer, ids_inner, uint32_t(outer * inner), inner, uint32_t(rows), id_bytes == 8 ? 1u : 0u},
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
