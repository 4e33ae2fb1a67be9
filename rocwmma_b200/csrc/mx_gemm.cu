// D = alpha * A * B + beta * C with both operands in a 4-bit block-scaled format (mx_format.cuh):
// A is m x k, B is k x n held as n rows of k, C and D are m x n, row-major.
//
// tcgen05.mma of the block-scaled kinds multiplies 64 values of K a step and applies the scales
// inside the tensor core; codes come by TMA in the 128-byte swizzle, scale tiles by TMA as they
// are stored and from shared memory to tensor memory by tcgen05.cp.  fp32 accumulation in tensor
// memory, one rounding to the output type after alpha and beta.
#include "common.cuh"
#include "mx_format.cuh"
#include "rocwmma/rocwmma_block.hpp"
#include "runtime.cuh"
#include "tile_schedule.cuh"
#include <cuda.h>

namespace b200wmma
{
    using namespace rocwmma::block;

    namespace
    {
        constexpr uint32_t SLOT_K      = 256; // values of K in a ring slot: one 128-byte row
        constexpr uint32_t MMA_K       = 64;
        constexpr uint32_t ROW_TILE    = 128;
        constexpr uint32_t CODE_BYTES  = ROW_TILE * 128;
        constexpr uint32_t NUM_THREADS = 192;
        constexpr uint32_t MAX_STAGES  = 8;
        constexpr uint32_t PREFETCH_SLOTS = 8; // of a block's stretch, requested into L2 ahead
        constexpr long long SETTLE_CYCLES = 2000000; // leaving early: copies in flight land

        struct Params
        {
            void const* c;
            void*       d;
            uint32_t    m, n, k, ldc, ldd;
            float       alpha, beta;
            uint32_t*   status;
        };

        template <ScaleKind KIND>
        constexpr uint32_t slotGroups() // scale tiles of 128 rows in a ring slot
        {
            return KIND == ScaleKind::E4M3_16 ? 4u : 2u;
        }

        // Loads and MMAs are issued by one thread each, whose instructions follow one another at four
        // or more cycles: a division by the ring's depth, or a descriptor put together anew, costs as
        // much as an MMA.  So slots are counted with a position that wraps, and descriptors are one
        // 32-bit sum (their upper halves never change).
        struct RingPosition
        {
            uint32_t slot = 0, phase = 0, offset = 0; // offset of the slot in shared memory
            __device__ void next(uint32_t stages, uint32_t slotBytes)
            {
                ++slot;
                offset += slotBytes;
                if(slot == stages)
                {
                    slot   = 0;
                    offset = 0;
                    phase ^= 1u;
                }
            }
        };
        __device__ inline uint64_t descAt(uint64_t base, uint32_t bytes)
        {
            return (base & 0xffffffff00000000ull) | (uint32_t(base) + (bytes >> 4));
        }

        // alpha and beta as everywhere in this library: a rounded product each, a rounded sum.
        template <typename OutT>
        __device__ inline OutT finish(float acc, float alpha, float beta, OutT const* c)
        {
            float r = __fmul_rn(alpha, acc);
            if(c)
                r = __fadd_rn(r, __fmul_rn(beta, toFloat(*c)));
            return fromFloat<OutT>(r);
        }

        __device__ inline void settle()
        {
            const long long start = clock64();
            while(clock64() - start < SETTLE_CYCLES)
            {
            }
        }

        // ---- thin products -----------------------------------------------------------------
        // One of m and n is small (a decoding batch; one token): the other operand, whose rows
        // are the MMA's M here, 128 to a block, streams from HBM once and bounds the call.  The
        // thin operand is the MMA's N, padded to 16 rows; its scales are one tile of 128.  A cluster of
        // `parts` blocks shares a tile, each a stretch of K, so that the stream comes through all SMs.
        // Every block puts its partial sums where its ring was, and adds up its share of the thin
        // rows out of the shared memory of the whole cluster, always in the order of the blocks.
        //
        // A block holds columns of tensor memory only while it needs nothing of another block: it gives
        // them back before it waits for its cluster.  tcgen05.alloc waits, without a limit, until its SM
        // has a contiguous range of that size, and how ranges are placed is the hardware's business; so
        // clusters that waited for each other's blocks with columns in hand could wait for good.
        // 1 x 8192 x 8192 MXF4: 9.1 us a call, 5.5 for its bytes; 64 x 16384 x 4096 NVF4: 12.0 and 6.
        // (With the sums sent to the block that adds them up, and the columns held until the end: 9.5 and 13.8;
        // 8192 x 64 x 2048 MXF4: 10.4 us so, 7.0 now.)
        constexpr uint32_t THIN_ROWS = 128; // at most, of the thin operand
        static_assert(THIN_ROWS <= MX_TILE_ROWS, "one scale tile to a ring slot's group");
        struct ThinParams
        {
            void const* c;
            void*       d;
            uint32_t    rows, thin, k; // rows of the streamed and of the thin operand
            uint64_t    cRow, cThin, dRow, dThin; // distance of neighbouring elements of C and D along each
            float       alpha, beta;
            uint32_t    nq, parts, stages, slotBytes, tmemCols;
            void const* r; // codes of the streamed operand, for requests ahead
            uint64_t    ldr;
            uint32_t*   status;
        };
        struct ThinControl
        {
            uint64_t   full[MAX_STAGES], empty[MAX_STAGES], accFull;
            AbortState abort;
            uint32_t   tmemBase;
        };

        __device__ inline float4 loadCluster4(uint32_t addr)
        {
            float4 v;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(addr)
                         : "memory");
            return v;
        }
        __device__ inline float loadCluster(uint32_t addr)
        {
            float v;
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
            return v;
        }

        // Four neighbouring elements of D, or the first `count` of them.  `wide`: D and C lie on the
        // boundary of four.
        template <typename OutT>
        __device__ inline void putFour(OutT* d, OutT const* c, ThinParams const& p, bool wide, uint32_t count, float4 acc)
        {
            struct alignas(4 * sizeof(OutT)) Four
            {
                OutT v[4];
            };
            const float a[4] = {acc.x, acc.y, acc.z, acc.w};
            if(wide && count >= 4u)
            {
                Four o;
                if(c)
                    o = *reinterpret_cast<Four const*>(c);
#pragma unroll
                for(int i = 0; i < 4; ++i)
                    o.v[i] = finish<OutT>(a[i], p.alpha, p.beta, c ? &o.v[i] : nullptr);
                *reinterpret_cast<Four*>(d) = o;
            }
            else
            {
#pragma unroll
                for(uint32_t i = 0; i < 4u; ++i)
                    if(i < count)
                        d[i] = finish<OutT>(a[i], p.alpha, p.beta, c ? c + i : nullptr);
            }
        }

        // The block's share of the thin rows, summed over the rings of the PARTS blocks of the cluster and
        // finished.  ring: shared-memory address of [thin row][row of the tile], the same in each.
        // A thread has eight loads in flight: one from another block's memory takes long.
        template <typename OutT, uint32_t PARTS>
        __device__ inline void finishShare(ThinParams const& p, uint32_t ring, uint32_t tile, uint32_t part)
        {
            constexpr uint32_t Q = 8u / PARTS; // thin rows at a time
            const uint32_t     share = p.nq / PARTS, first = part * share; // thin row
            const uint32_t     mine  = first < p.thin ? min(share, p.thin - first) : 0u;
            const uint64_t     row0  = uint64_t(tile) * ROW_TILE;
            const uint32_t     left  = uint32_t(min(uint64_t(ROW_TILE), p.rows - row0));
            OutT*              d     = static_cast<OutT*>(p.d) + row0 * p.dRow + first * p.dThin;
            OutT const*        c     = p.c ? static_cast<OutT const*>(p.c) + row0 * p.cRow + first * p.cThin : nullptr;
            uint32_t           from[PARTS];
#pragma unroll
            for(uint32_t o = 0; o < PARTS; ++o)
                from[o] = (PARTS > 1u ? map_to_cta(ring, o) : ring) + first * ROW_TILE * 4u;
            if(p.dRow == 1u)
            {
                // a warp takes a row of D, a lane four columns
                constexpr uint32_t WARPS = NUM_THREADS / 32u;
                const uint32_t     warp = threadIdx.x / 32u, r = 4u * (threadIdx.x % 32u);
                if(r >= left)
                    return;
                d += r;
                c = c ? c + r : nullptr;
                for(uint32_t q0 = warp; q0 < mine; q0 += Q * WARPS)
                {
                    float4 v[Q][PARTS];
#pragma unroll
                    for(uint32_t i = 0; i < Q; ++i)
#pragma unroll
                        for(uint32_t o = 0; o < PARTS; ++o)
                            if(q0 + i * WARPS < mine)
                                v[i][o] = loadCluster4(from[o] + ((q0 + i * WARPS) * ROW_TILE + r) * 4u);
#pragma unroll
                    for(uint32_t i = 0; i < Q; ++i)
                    {
                        const uint32_t q = q0 + i * WARPS;
                        if(q >= mine)
                            break;
                        float4 acc = v[i][0];
#pragma unroll
                        for(uint32_t o = 1; o < PARTS; ++o)
                        {
                            acc.x += v[i][o].x;
                            acc.y += v[i][o].y;
                            acc.z += v[i][o].z;
                            acc.w += v[i][o].w;
                        }
                        putFour<OutT>(d + q * p.dThin, c ? c + q * p.cThin : nullptr, p, true, left - r, acc);
                    }
                }
            }
            else if(threadIdx.x < left)
            {
                // a thread takes a row of D, four columns at a time
                const uint32_t r = threadIdx.x;
                d += r * p.dRow;
                c = c ? c + r * p.cRow : nullptr;
                for(uint32_t q0 = 0; q0 < mine; q0 += 4u)
                {
                    float v[4][PARTS], acc[4];
#pragma unroll
                    for(uint32_t i = 0; i < 4u; ++i)
#pragma unroll
                        for(uint32_t o = 0; o < PARTS; ++o)
                            v[i][o] = q0 + i < mine ? loadCluster(from[o] + ((q0 + i) * ROW_TILE + r) * 4u) : 0.0f;
#pragma unroll
                    for(uint32_t i = 0; i < 4u; ++i)
                    {
                        acc[i] = v[i][0];
#pragma unroll
                        for(uint32_t o = 1; o < PARTS; ++o)
                            acc[i] += v[i][o];
                    }
                    putFour<OutT>(d + q0, c ? c + q0 : nullptr, p, first % 4u == 0u, mine - q0,
                                  make_float4(acc[0], acc[1], acc[2], acc[3]));
                }
            }
        }

        template <ScaleKind KIND, typename OutT>
        __global__ void __launch_bounds__(NUM_THREADS)
            mxGemmThinKernel(const __grid_constant__ CUtensorMap mapR,
                             const __grid_constant__ CUtensorMap mapQ,
                             const __grid_constant__ CUtensorMap mapScaleR,
                             const __grid_constant__ CUtensorMap mapScaleQ, const ThinParams p)
        {
            constexpr uint32_t GROUPS = slotGroups<KIND>();
            extern __shared__ uint8_t smemRaw[];
            uint8_t*     ring = smemRaw + ((1024u - (smem_addr(smemRaw) & 1023u)) & 1023u);
            ThinControl* ctl  = reinterpret_cast<ThinControl*>(ring + p.stages * p.slotBytes);

            const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
            const uint32_t tile = blockIdx.x / p.parts, part = blockIdx.x % p.parts; // part: rank in the cluster
            const uint32_t allSlots = (p.k + SLOT_K - 1) / SLOT_K;
            const uint32_t slot0 = uint32_t(uint64_t(part) * allSlots / p.parts);
            const uint32_t numSlots = uint32_t(uint64_t(part + 1u) * allSlots / p.parts) - slot0;
            const uint32_t qBytes   = p.nq * 128u;

            if(threadIdx.x == 0)
            {
                for(uint32_t s = 0; s < p.stages; ++s)
                {
                    mbar_init(&ctl->full[s], 1);
                    mbar_init(&ctl->empty[s], 1);
                }
                mbar_init(&ctl->accFull, 1);
                ctl->abort.flag = 0;
                ctl->abort.code = 0;
                mbar_init_fence();
                tma_prefetch_descriptor(&mapR);
                tma_prefetch_descriptor(&mapQ);
                tma_prefetch_descriptor(&mapScaleR);
                tma_prefetch_descriptor(&mapScaleQ);
            }
            else if(warp >= 2u)
            {
                // The streamed operand's first slots are requested into L2 while the previous
                // kernel of the stream (often the quantisation of the thin operand) still runs: a
                // request reads nothing into the SM, and L2 is where a late write would land too.
                // (Not by TMA: the loads would queue up behind the requests, 1 us for 16 slots.)
                const uint64_t row = uint64_t(tile) * ROW_TILE + threadIdx.x - 64u;
                if(row < p.rows)
                    for(uint32_t it = 0; it < numSlots && it < PREFETCH_SLOTS; ++it)
                    {
                        const uint64_t at = uint64_t(slot0 + it) * 128u;
                        if(at * 2u < p.k)
                            prefetch_l2(static_cast<uint8_t const*>(p.r) + row * p.ldr + at);
                    }
            }
            __syncwarp();
            if(warp == 1)
            {
                tmem_alloc(&ctl->tmemBase, p.tmemCols);
                tmem_relinquish_alloc_permit();
            }
            tc_fence_before_sync();
            __syncthreads();
            tc_fence_after_sync();
            const uint32_t tmem = ctl->tmemBase;
            grid_dependency_wait();
            grid_launch_dependents();

            if(warp == 0)
            {
                if(elect_one())
                {
                    RingPosition at;
                    int32_t      x = int32_t(slot0 * 128u), group = int32_t(slot0 * GROUPS);
                    for(uint32_t it = 0; it < numSlots; ++it, x += 128, group += int32_t(GROUPS))
                    {
                        uint64_t* full = &ctl->full[at.slot];
                        if(!mbar_wait(&ctl->empty[at.slot], at.phase ^ 1u, &ctl->abort, WAIT_STAGE_EMPTY))
                        {
                            settle();
                            break;
                        }
                        uint8_t* slot = ring + at.offset;
                        mbar_expect_tx(full, p.slotBytes);
                        tma_load_2d(slot, &mapR, full, x, int32_t(tile * ROW_TILE));
                        tma_load_2d(slot + CODE_BYTES, &mapQ, full, x, 0);
                        tma_load_3d(slot + CODE_BYTES + qBytes, &mapScaleR, full, 0, group, int32_t(tile));
                        tma_load_3d(slot + CODE_BYTES + qBytes + GROUPS * MX_TILE_BYTES, &mapScaleQ, full, 0, group, 0);
                        at.next(p.stages, p.slotBytes);
                    }
                }
            }
            else if(warp == 1)
            {
                if(elect_one())
                {
                    // accumulator, then the scales of two ring slots in turn
                    const uint32_t scaleCols = 4u * GROUPS * 2u;
                    uint32_t       scale = tmem + (p.nq + 31u) / 32u * 32u, otherScale = scale + scaleCols;
                    const uint32_t base  = smem_addr(ring);
                    const uint64_t descR = smem_desc_kmajor_sw128(base), descQ = descAt(descR, CODE_BYTES);
                    const uint64_t descS = smem_desc_scales(base + CODE_BYTES + qBytes);
                    const uint32_t idesc = make_instr_desc_scaled(KIND, ROW_TILE, p.nq, 0);
                    RingPosition   at;
                    uint32_t       left = p.k - slot0 * SLOT_K, more = 0;
                    bool           ok = true;
                    for(uint32_t it = 0; it < numSlots; ++it, left -= SLOT_K)
                    {
                        if(!mbar_wait(&ctl->full[at.slot], at.phase, &ctl->abort, WAIT_STAGE_FULL))
                        {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                        const uint64_t dS = descAt(descS, at.offset);
#pragma unroll
                        for(uint32_t g = 0; g < GROUPS; ++g)
                        {
                            tmem_copy_scales(scale + 4u * g, descAt(dS, g * MX_TILE_BYTES));
                            tmem_copy_scales(scale + 4u * (GROUPS + g), descAt(dS, (GROUPS + g) * MX_TILE_BYTES));
                        }
                        const uint64_t dR = descAt(descR, at.offset), dQ = descAt(descQ, at.offset);
                        auto step = [&](uint32_t ks) {
                            // MXF4 takes a tile's four scales in two steps, NVF4 in one
                            const uint32_t g  = KIND == ScaleKind::E4M3_16 ? ks : ks / 2u;
                            const uint32_t id = KIND == ScaleKind::E4M3_16 ? 0u : (ks & 1u) * 2u;
                            mma_scaled<KIND>(tmem, descAt(dR, ks * 32u), descAt(dQ, ks * 32u), idesc | id << 4 | id << 29,
                                             scale + 4u * g, scale + 4u * (GROUPS + g), more);
                            more = 1;
                        };
                        if(left >= SLOT_K)
                        {
#pragma unroll
                            for(uint32_t ks = 0; ks < SLOT_K / MMA_K; ++ks)
                                step(ks);
                        }
                        else
                            for(uint32_t ks = 0; ks * MMA_K < left; ++ks)
                                step(ks);
                        mma_commit(&ctl->empty[at.slot]);
                        const uint32_t swap = scale;
                        scale               = otherScale;
                        otherScale          = swap;
                        at.next(p.stages, p.slotBytes);
                    }
                    if(ok)
                        mma_commit(&ctl->accFull);
                }
            }

            // The sums go where the ring was, as [thin row][row of the tile] (a lane has a row of the tile,
            // registers hold thin rows), the columns back to the SM, and only then the block waits
            // for its cluster.
            const bool drains = warp >= 2u;
            bool       ready  = false;
            if(drains)
                ready = mbar_wait_warp(&ctl->accFull, 0, &ctl->abort, WAIT_ACC_FULL); // the last slot has been read
            if(drains && ready)
            {
                tc_fence_after_sync();
                const uint32_t inTile = warp % 4u * 32u + lane, taddr = tmem + ((warp % 4u * 32u) << 16);
                uint32_t*      at     = reinterpret_cast<uint32_t*>(ring) + inTile;
                for(uint32_t q0 = 0; q0 < p.nq; q0 += 16u)
                {
                    uint32_t raw[16];
                    tmem_load_32x32b_x16(taddr + q0, raw);
                    tmem_load_wait();
#pragma unroll
                    for(uint32_t j = 0; j < 16u; ++j)
                        at[(q0 + j) * ROW_TILE] = raw[j];
                }
            }
            tc_fence_before_sync();
            __syncthreads();
            if(warp == 1)
            {
                __syncwarp();
                tc_fence_after_sync();
                tmem_dealloc(tmem, p.tmemCols);
            }
            __syncwarp();
            if(p.parts > 1u)
                cluster_sync();
            switch(p.parts)
            {
            case 1:
                finishShare<OutT, 1>(p, smem_addr(ring), tile, part);
                break;
            case 2:
                finishShare<OutT, 2>(p, smem_addr(ring), tile, part);
                break;
            case 4:
                finishShare<OutT, 4>(p, smem_addr(ring), tile, part);
                break;
            default:
                finishShare<OutT, 8>(p, smem_addr(ring), tile, part);
            }
            __syncwarp();
            if(p.parts > 1u)
            {
                // no block leaves while another may still read its sums (what this one has read has arrived:
                // it has been stored)
                cluster_arrive_relaxed();
                cluster_wait();
            }
            if(threadIdx.x == 0 && ctl->abort.flag != 0u && p.status != nullptr)
            {
                atomicExch(&p.status[1], ctl->abort.code);
                atomicExch(&p.status[0], 1u);
            }
        }

        // ---- large products: CTA pairs -----------------------------------------------------
        // A pair of blocks owns a 256 x 256 tile (cta_group::2): each stages its own 128 rows of
        // A and half of the columns of B, the scales of its rows of A and those of all of B; the
        // even block issues MMAs of M = 256.  Persistent; warp 0 loads, warp 1 multiplies, warps 2
        // to 9 drain, warp 10 moves boxes of C and D.
        //
        // Tensor memory has 512 columns: two accumulators of 256 would leave none for the scales.
        // So the two overlap: the second starts at column ACC1, the scales of two ring slots lie
        // behind it, and the first MMA of a tile waits only until the tile before has drained the
        // columns that both accumulators share, which are drained first.
        // 8192 x 8192 x 8192 MXF4: 182 us (6.0 PFLOP/s) in bursts, 216 under the power limit.  One tile to
        // a pair, 1000 x 4100 x 4111 NVF4 with C: 19 us, of which the MMAs take 7.
        constexpr uint32_t P_TILE      = 256;
        // With C, whose boxes come from memory, twice the boxes are worth more than a fifth slot: one
        // 256 x 256 tile f32 is drained in 5.8 us instead of 8.3, its MMAs take 0.1 us longer.
        constexpr uint32_t P_STAGES    = 5, P_STAGES_C = 4;
        constexpr uint32_t BOX_BYTES   = 128 * 64; // 128 rows x 64 bytes of D (or C)
        constexpr uint32_t BOXES = 4, BOXES_C = 8;
        constexpr uint32_t P_THREADS   = 352;
        constexpr uint32_t DRAIN_WARPS = 8;

        struct PairParams
        {
            void const* c;
            void*       d;
            uint32_t    m, n, k, ldc, ldd;
            float       alpha, beta;
            uint32_t    band, stages, boxes;
            uint32_t*   status;
        };
        struct PairControl
        {
            uint64_t   full[P_STAGES], empty[P_STAGES], accFull[2], accShared;
            uint64_t   cFull[BOXES_C], boxFull[BOXES_C], boxFree[BOXES_C];
            AbortState abort;
            uint32_t   tmemBase;
        };
        template <ScaleKind KIND>
        constexpr uint32_t pairSlotBytes()
        {
            return 2u * CODE_BYTES + 3u * slotGroups<KIND>() * MX_TILE_BYTES;
        }
        // (Large enough that no block of the thin kernel fits beside it, which would leave it waiting for
        // columns.)
        template <ScaleKind KIND>
        constexpr uint32_t pairSmemBytes(bool useC)
        {
            return 1024u + (useC ? P_STAGES_C : P_STAGES) * pairSlotBytes<KIND>() + (useC ? BOXES_C : BOXES) * BOX_BYTES
                   + uint32_t(sizeof(PairControl));
        }

        // The boxes of one tile, 128 rows x 64 bytes of D each, in the order in which they are drained:
        // from column `first` on, around the tile's end.  Those that hold a whole number of 16-byte
        // pieces of D pass through shared memory (`staged`); one that D's last column cuts inside a
        // piece is stored by the draining threads.
        template <typename OutT>
        struct Boxes
        {
            static constexpr uint32_t COLS  = 64 / sizeof(OutT);
            static constexpr uint32_t VEC   = 16 / sizeof(OutT);
            static constexpr uint32_t COUNT = P_TILE / COLS;
            uint32_t first, left, valid, ragged;
            __device__ Boxes(PairParams const& p, uint32_t col0, uint32_t firstCol)
                : first(firstCol / COLS), left(p.n - col0), valid(min(COUNT, (left + COLS - 1u) / COLS)),
                  ragged(left < P_TILE && left % VEC != 0u ? valid - 1u : COUNT)
            {
            }
            __device__ uint32_t at(uint32_t i) const
            {
                return (first + i) % COUNT;
            }
            __device__ bool staged(uint32_t box) const
            {
                return box < valid && box != ragged;
            }
        };

        // Warp 10, one thread: boxes of D go out by TMA as the draining warps fill them; with C, boxes
        // of it come in by TMA to where D's will be, as many ahead as there are boxes.
        template <typename OutT>
        __device__ inline bool moveBoxes(PairControl* ctl, uint8_t* staging, CUtensorMap const* mapC, CUtensorMap const* mapD,
                                         PairParams const& p, uint32_t first, uint32_t row0, uint32_t col0, uint32_t& count)
        {
            using B                = Boxes<OutT>;
            constexpr uint32_t LAG = 2;
            const B            boxes(p, col0, first);
            const bool         useC = p.c != nullptr;
            uint32_t   asked = 0, askedCount = count;
            auto       askForC = [&] {
                while(asked < B::COUNT && !boxes.staged(boxes.at(asked)))
                    ++asked;
                if(asked == B::COUNT)
                    return;
                const uint32_t b = askedCount & (p.boxes - 1u);
                mbar_expect_tx(&ctl->cFull[b], BOX_BYTES);
                tma_load_2d(staging + b * BOX_BYTES, mapC, &ctl->cFull[b], int32_t(col0 + boxes.at(asked) * B::COLS), int32_t(row0));
                ++asked;
                ++askedCount;
            };
            if(useC) // the boxes of the tile before have been read out
                for(uint32_t b = 0; b < p.boxes; ++b)
                    askForC();
            for(uint32_t i = 0; i < B::COUNT; ++i)
            {
                const uint32_t box = boxes.at(i);
                if(!boxes.staged(box))
                    continue;
                const uint32_t b = count & (p.boxes - 1u);
                if(!mbar_wait(&ctl->boxFull[b], (count & p.boxes) != 0u, &ctl->abort, WAIT_ACC_FULL))
                    return false;
                tma_store_2d(mapD, staging + b * BOX_BYTES, int32_t(col0 + box * B::COLS), int32_t(row0));
                tma_store_commit();
                // The store two before has been read out.  (Waiting for the one just issued would make
                // every box as long as a store takes to read its source, 0.4 us.)
                tma_store_wait_read<LAG>();
                if(useC)
                {
                    if(askedCount + LAG <= count + p.boxes)
                        askForC();
                }
                else if(count >= LAG)
                    mbar_arrive(&ctl->boxFree[(count - LAG) & (p.boxes - 1u)]);
                ++count;
            }
            if(useC)
                tma_store_wait_read<0>();
            return true;
        }

        // Drains one tile's accumulator: TMEM -> registers -> shared memory in the TMA's 64-byte
        // swizzle, in place of C's box where there is one.  Two sets of four warps take boxes in
        // turn.  (Four warps, with one of their threads moving the boxes as well: 4.7 us for the last
        // tile of 256 columns bf16, 11 us f32 with C; so: 3.0 and 5.8.)
        template <typename OutT, bool C>
        __device__ inline bool drainTile(PairControl* ctl, uint8_t* staging, PairParams const& p, uint32_t taddr, uint32_t set,
                                         uint32_t first, uint32_t shared, uint32_t accBar, uint32_t accPhase, uint32_t row0,
                                         uint32_t rowIn, uint32_t col0, uint32_t& count, uint32_t leaderShared)
        {
            using B = Boxes<OutT>;
            constexpr uint32_t COLS = B::COLS, VEC = B::VEC;
            const B            boxes(p, col0, first);
            const uint32_t     row = row0 + rowIn, lastShared = shared / COLS - 1u - (shared / COLS - 1u + set) % 2u;
            if constexpr(C)
            {
                // the row's part of C into L2 while the tile is multiplied
                if(row < p.m)
                {
                    uint8_t const* c = static_cast<uint8_t const*>(p.c) + (uint64_t(row) * p.ldc + col0) * sizeof(OutT);
                    const uint32_t bytes = min(P_TILE, boxes.left) * uint32_t(sizeof(OutT));
                    for(uint32_t at = set * 128u; at < bytes; at += 256u)
                        prefetch_l2(c + at);
                }
            }
            if(!mbar_wait_warp(&ctl->accFull[accBar], accPhase, &ctl->abort, WAIT_ACC_FULL))
                return false;
            tc_fence_after_sync();
#pragma unroll 1
            for(uint32_t i = 0; i < B::COUNT; ++i)
            {
                const uint32_t box = boxes.at(i), mine = count;
                count += boxes.staged(box) ? 1u : 0u;
                if(i % 2u != set)
                    continue;
                uint32_t raw[COLS];
                if(box < boxes.valid)
                {
                    if constexpr(COLS == 32)
                        tmem_load_32x32b_x32(taddr + box * COLS, raw);
                    else
                        tmem_load_32x32b_x16(taddr + box * COLS, raw);
                    tmem_load_wait();
                }
                if(i == lastShared)
                {
                    // this warp's part of the columns that the next tile's accumulator shares is out
                    tc_fence_before_sync();
                    if(rowIn % 32u == 0u)
                        mbar_arrive_cluster(leaderShared);
                }
                if(box >= boxes.valid)
                    continue;
                if(box == boxes.ragged)
                {
#pragma unroll
                    for(uint32_t e = 0; e < COLS; ++e)
                        if(row < p.m && box * COLS + e < boxes.left)
                        {
                            const uint64_t col = col0 + box * COLS + e;
                            OutT const*    c   = C ? static_cast<OutT const*>(p.c) + uint64_t(row) * p.ldc + col : nullptr;
                            static_cast<OutT*>(p.d)[uint64_t(row) * p.ldd + col]
                                = finish<OutT>(__uint_as_float(raw[e]), p.alpha, p.beta, c);
                        }
                    continue;
                }
                const uint32_t b = mine & (p.boxes - 1u), use = (mine & p.boxes) != 0u;
                const bool     open = C ? mbar_wait_warp(&ctl->cFull[b], use, &ctl->abort, WAIT_STAGE_FULL)
                                        : mbar_wait_warp(&ctl->boxFree[b], use ^ 1u, &ctl->abort, WAIT_DRAIN);
                if(!open)
                    return false;
                uint8_t* at = staging + b * BOX_BYTES + rowIn * 64u;
#pragma unroll
                for(uint32_t ch = 0; ch < 4u; ++ch)
                {
                    // 64-byte swizzle: piece index ^ (row / 2 % 4)
                    uint4* piece = reinterpret_cast<uint4*>(at + ((ch ^ ((rowIn >> 1) & 3u)) << 4));
                    alignas(16) OutT v[VEC];
                    if constexpr(C)
                        *reinterpret_cast<uint4*>(v) = *piece;
#pragma unroll
                    for(uint32_t e = 0; e < VEC; ++e)
                        v[e] = finish<OutT>(__uint_as_float(raw[ch * VEC + e]), p.alpha, p.beta, C ? &v[e] : nullptr);
                    *piece = *reinterpret_cast<uint4 const*>(v);
                }
                fence_async_shared();
                __syncwarp();
                if(rowIn % 32u == 0u)
                    mbar_arrive(&ctl->boxFull[b]);
            }
            return true;
        }

        template <ScaleKind KIND, typename OutT>
        __global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P_THREADS, 1)
            mxGemmPairKernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                             const __grid_constant__ CUtensorMap mapScaleA,
                             const __grid_constant__ CUtensorMap mapScaleB,
                             const __grid_constant__ CUtensorMap mapC, const __grid_constant__ CUtensorMap mapD,
                             const PairParams p)
        {
            constexpr uint32_t GROUPS     = slotGroups<KIND>();
            constexpr uint32_t SLOT       = pairSlotBytes<KIND>();
            constexpr uint32_t SCALE_COLS = 12u * GROUPS; // of one slot: 4 for A, 8 for B, a group
            constexpr uint32_t SHARED     = KIND == ScaleKind::E4M3_16 ? 96u : 64u;
            constexpr uint32_t ACC1       = 256u - SHARED;
            static_assert(ACC1 + 256u + 2u * SCALE_COLS <= 512u, "tensor memory");
            extern __shared__ uint8_t smemRaw[];
            uint8_t*       ring    = smemRaw + ((1024u - (smem_addr(smemRaw) & 1023u)) & 1023u);
            uint8_t*       staging = ring + p.stages * SLOT;
            PairControl*   ctl     = reinterpret_cast<PairControl*>(staging + p.boxes * BOX_BYTES);
            const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
            const uint32_t rank = cluster_cta_rank(), pairId = blockIdx.x / 2, pairs = gridDim.x / 2;
            const uint32_t numSlots = (p.k + SLOT_K - 1) / SLOT_K;
            const TileSchedule sched{(p.m + P_TILE - 1u) / P_TILE, (p.n + P_TILE - 1u) / P_TILE, 0u, P_TILE, 0u, p.band, pairs, 1u};

            if(threadIdx.x == 0)
            {
                for(uint32_t s = 0; s < p.stages; ++s)
                {
                    mbar_init(&ctl->full[s], 1);
                    mbar_init(&ctl->empty[s], 1);
                }
                for(uint32_t b = 0; b < 2u; ++b)
                    mbar_init(&ctl->accFull[b], 1);
                mbar_init(&ctl->accShared, 2u * DRAIN_WARPS);
                for(uint32_t b = 0; b < p.boxes; ++b)
                {
                    mbar_init(&ctl->cFull[b], 1);
                    mbar_init(&ctl->boxFull[b], DRAIN_WARPS / 2u);
                    mbar_init(&ctl->boxFree[b], 1);
                }
                ctl->abort.flag = 0;
                ctl->abort.code = 0;
                mbar_init_fence();
                tma_prefetch_descriptor(&mapA);
                tma_prefetch_descriptor(&mapB);
                tma_prefetch_descriptor(&mapScaleA);
                tma_prefetch_descriptor(&mapScaleB);
                tma_prefetch_descriptor(&mapD);
            }
            __syncwarp();
            cluster_arrive_relaxed();
            if(warp == 1)
            {
                tmem_alloc_pair(&ctl->tmemBase, 512);
                tmem_relinquish_alloc_permit_pair();
            }
            tc_fence_before_sync();
            __syncthreads();
            cluster_wait(); // both blocks' barriers exist before anything signals them remotely
            tc_fence_after_sync();
            const uint32_t tmem = ctl->tmemBase;
            grid_dependency_wait();
            grid_launch_dependents();

            uint32_t tm, col0, width;
            if(warp == 0)
            {
                if(elect_one())
                {
                    const uint32_t leaderFull = map_to_cta(smem_addr(&ctl->full[0]), 0);
                    RingPosition   at;
                    bool           ok = true;
                    for(uint32_t i = 0; ok && sched.get(pairId, i, tm, col0, width); ++i)
                    {
                        const int32_t rowA = int32_t(tm * P_TILE + rank * 128u), rowB = int32_t(col0 + rank * 128u);
                        const int32_t tileA = int32_t(tm * 2u + rank), tileB = int32_t(col0 / 128u);
                        int32_t       x = 0, group = 0;
                        for(uint32_t kb = 0; kb < numSlots; ++kb, x += 128, group += int32_t(GROUPS))
                        {
                            if(!mbar_wait(&ctl->empty[at.slot], at.phase ^ 1u, &ctl->abort, WAIT_STAGE_EMPTY))
                            {
                                ok = false;
                                break;
                            }
                            uint8_t*       slot = ring + at.offset;
                            const uint32_t full = leaderFull + at.slot * 8u;
                            if(rank == 0)
                                mbar_expect_tx(&ctl->full[at.slot], 2u * SLOT); // both blocks
                            tma_load_2d_pair(slot, &mapA, full, x, rowA);
                            tma_load_2d_pair(slot + CODE_BYTES, &mapB, full, x, rowB);
                            tma_load_3d_pair(slot + 2u * CODE_BYTES, &mapScaleA, full, 0, group, tileA);
                            tma_load_3d_pair(slot + 2u * CODE_BYTES + GROUPS * MX_TILE_BYTES, &mapScaleB, full, 0, group,
                                             tileB);
                            at.next(p.stages, SLOT);
                        }
                    }
                    if(!ok)
                        settle();
                }
            }
            else if(warp == 1)
            {
                if(rank == 0 && elect_one())
                {
                    const uint32_t base  = smem_addr(ring);
                    const uint64_t descA = smem_desc_kmajor_sw128(base), descB = descAt(descA, CODE_BYTES);
                    const uint64_t descS = smem_desc_scales(base + 2u * CODE_BYTES);
                    uint32_t       scale = tmem + 512u - SCALE_COLS, otherScale = scale - SCALE_COLS;
                    RingPosition   at;
                    bool           ok = true;
                    for(uint32_t i = 0; ok && sched.get(pairId, i, tm, col0, width); ++i)
                    {
                        // tile i - 1 has drained the columns that its accumulator shares with this one's
                        if(i > 0u && !mbar_wait(&ctl->accShared, (i - 1u) & 1u, &ctl->abort, WAIT_ACC_EMPTY))
                            break;
                        tc_fence_after_sync();
                        const uint32_t acc  = tmem + (i & 1u) * ACC1;
                        uint32_t       left = p.k, more = 0;
                        for(uint32_t kb = 0; kb < numSlots; ++kb, left -= SLOT_K)
                        {
                            if(!mbar_wait(&ctl->full[at.slot], at.phase, &ctl->abort, WAIT_STAGE_FULL))
                            {
                                ok = false;
                                break;
                            }
                            tc_fence_after_sync();
                            const uint64_t dS = descAt(descS, at.offset);
#pragma unroll
                            for(uint32_t g = 0; g < GROUPS; ++g)
                            {
                                tmem_copy_scales_pair(scale + 4u * g, descAt(dS, g * MX_TILE_BYTES));
                                tmem_copy_scales_pair(scale + 4u * GROUPS + 8u * g, descAt(dS, (GROUPS + g) * MX_TILE_BYTES));
                                tmem_copy_scales_pair(scale + 4u * GROUPS + 8u * g + 4u,
                                                      descAt(dS, (2u * GROUPS + g) * MX_TILE_BYTES));
                            }
                            const uint64_t dA = descAt(descA, at.offset), dB = descAt(descB, at.offset);
                            auto           step = [&](uint32_t ks) {
                                const uint32_t g  = KIND == ScaleKind::E4M3_16 ? ks : ks / 2u;
                                const uint32_t id = KIND == ScaleKind::E4M3_16 ? 0u : (ks & 1u) * 2u;
                                mma_scaled_pair<KIND>(acc, descAt(dA, ks * 32u), descAt(dB, ks * 32u),
                                                      make_instr_desc_scaled(KIND, 256u, P_TILE, id), scale + 4u * g,
                                                      scale + 4u * GROUPS + 8u * g, more);
                                more = 1;
                            };
                            if(left >= SLOT_K)
                            {
#pragma unroll
                                for(uint32_t ks = 0; ks < SLOT_K / MMA_K; ++ks)
                                    step(ks);
                            }
                            else
                                for(uint32_t ks = 0; ks * MMA_K < left; ++ks)
                                    step(ks);
                            mma_commit_pair(&ctl->empty[at.slot], 0x3);
                            const uint32_t swap = scale;
                            scale               = otherScale;
                            otherScale          = swap;
                            at.next(p.stages, SLOT);
                        }
                        if(ok)
                            mma_commit_pair(&ctl->accFull[i & 1u], 0x3);
                    }
                }
            }
            else if(warp < 2u + DRAIN_WARPS)
            {
                const uint32_t quad = warp % 4, rowIn = quad * 32u + lane, set = (warp - 2u) / 4u;
                const uint32_t leaderShared = map_to_cta(smem_addr(&ctl->accShared), 0);
                uint32_t       count = 0;
                bool           ok    = true;
                for(uint32_t i = 0; ok && sched.get(pairId, i, tm, col0, width); ++i)
                {
                    // the second accumulator's shared columns are its first ones, the first one's its last
                    const uint32_t buf = i & 1u, taddr = tmem + ((quad * 32u) << 16) + buf * ACC1;
                    const uint32_t first = buf ? 0u : ACC1, row0 = tm * P_TILE + rank * 128u;
                    ok = p.c ? drainTile<OutT, true>(ctl, staging, p, taddr, set, first, SHARED, buf, (i >> 1) & 1u, row0, rowIn,
                                                     col0, count, leaderShared)
                             : drainTile<OutT, false>(ctl, staging, p, taddr, set, first, SHARED, buf, (i >> 1) & 1u, row0, rowIn,
                                                      col0, count, leaderShared);
                }
            }
            else if(elect_one())
            {
                uint32_t count = 0;
                bool     ok    = true;
                for(uint32_t i = 0; ok && sched.get(pairId, i, tm, col0, width); ++i)
                    ok = moveBoxes<OutT>(ctl, staging, &mapC, &mapD, p, i & 1u ? 0u : ACC1, tm * P_TILE + rank * 128u, col0, count);
                if(!ok)
                    settle();
                tma_store_wait_read<0>(); // shared memory outlives the stores' reads of it
            }

            tc_fence_before_sync();
            __syncthreads();
            cluster_arrive_relaxed(); // neither block leaves while the other may still signal it
            cluster_wait();
            if(warp == 1)
            {
                __syncwarp();
                tc_fence_after_sync();
                tmem_dealloc_pair(tmem, 512);
            }
            if(threadIdx.x == 0 && ctl->abort.flag != 0u && p.status != nullptr)
            {
                atomicExch(&p.status[1], ctl->abort.code);
                atomicExch(&p.status[0], 1u);
            }
        }

        // ---- host side -------------------------------------------------------------------
        int codeMap(CUtensorMap* map, void const* codes, uint32_t rows, uint32_t k, uint64_t ld, uint32_t boxRows)
        {
            const cuuint64_t dims[2]    = {(cuuint64_t(k) + 1) / 2, rows};
            const cuuint64_t strides[1] = {ld};
            const cuuint32_t box[2]     = {128, boxRows};
            const cuuint32_t estr[2]    = {1, 1};
            EncodeFn         fn         = tensorMapEncoder();
            if(!fn)
                return B200WMMA_ERR_CUDA;
            const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims,
                                  strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            return r == CUDA_SUCCESS ? B200WMMA_OK : B200WMMA_ERR_CUDA;
        }

        // Scale tiles as [row tiles][groups][128 words]; box: the groups of a ring slot.
        int scaleMap(CUtensorMap* map, void const* scales, uint32_t rows, uint32_t groups,
                     uint32_t boxGroups, uint32_t boxTiles)
        {
            const cuuint64_t dims[3]    = {128, groups, mxRowTiles(rows)};
            const cuuint64_t strides[2] = {MX_TILE_BYTES, cuuint64_t(groups) * MX_TILE_BYTES};
            const cuuint32_t box[3]     = {128, boxGroups, boxTiles};
            const cuuint32_t estr[3]    = {1, 1, 1};
            EncodeFn         fn         = tensorMapEncoder();
            if(!fn)
                return B200WMMA_ERR_CUDA;
            const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(scales), dims,
                                  strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            return r == CUDA_SUCCESS ? B200WMMA_OK : B200WMMA_ERR_CUDA;
        }

        // Rows of C or D; box: 128 rows x 64 bytes.
        template <typename OutT>
        int outputMap(CUtensorMap* map, void const* base, uint32_t rows, uint32_t cols, uint32_t ld)
        {
            const cuuint64_t dims[2]    = {cols, rows};
            const cuuint64_t strides[1] = {cuuint64_t(ld) * sizeof(OutT)};
            const cuuint32_t box[2]     = {cuuint32_t(64 / sizeof(OutT)), 128};
            const cuuint32_t estr[2]    = {1, 1};
            EncodeFn         fn         = tensorMapEncoder();
            if(!fn)
                return B200WMMA_ERR_CUDA;
            const CUtensorMapDataType type = sizeof(OutT) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                             : std::is_same<OutT, __half>::value
                                                 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
            const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            return r == CUDA_SUCCESS ? B200WMMA_OK : B200WMMA_ERR_CUDA;
        }

        struct Operands
        {
            void const *a, *aScales, *b, *bScales;
            uint64_t    lda, ldb;
        };

        template <ScaleKind KIND, typename OutT>
        int launchPairs(Operands const& o, Params const& q, int sms, cudaStream_t stream)
        {
            constexpr uint32_t GROUPS = slotGroups<KIND>();
            const uint32_t     groups = mxGroups(KIND == ScaleKind::E4M3_16, q.k);
            const uint64_t     tiles  = uint64_t((q.m + P_TILE - 1u) / P_TILE) * ((q.n + P_TILE - 1u) / P_TILE);
            if(tiles > 0x7fffffffull)
                return B200WMMA_ERR_TOO_LARGE;
            CUtensorMap mapA, mapB, mapScaleA, mapScaleB, mapC, mapD;
            int         rc = codeMap(&mapA, o.a, q.m, q.k, o.lda, 128);
            if(rc == B200WMMA_OK)
                rc = codeMap(&mapB, o.b, q.n, q.k, o.ldb, 128);
            if(rc == B200WMMA_OK)
                rc = scaleMap(&mapScaleA, o.aScales, q.m, groups, GROUPS, 1);
            if(rc == B200WMMA_OK)
                rc = scaleMap(&mapScaleB, o.bScales, q.n, groups, GROUPS, 2);
            if(rc == B200WMMA_OK)
                rc = outputMap<OutT>(&mapD, q.d, q.m, q.n, q.ldd);
            mapC = mapD;
            if(rc == B200WMMA_OK && q.c)
                rc = outputMap<OutT>(&mapC, q.c, q.m, q.n, q.ldc);
            if(rc != B200WMMA_OK)
                return rc;
            static_assert(pairSmemBytes<KIND>(true) >= 200u * 1024u && pairSmemBytes<KIND>(false) >= 200u * 1024u,
                          "a thin block, 28 KB or more, must not fit beside a pair's");
            const uint32_t  smem = pairSmemBytes<KIND>(q.c != nullptr);
            static uint32_t done[64] = {};
            rc = optInSharedMemory(mxGemmPairKernel<KIND, OutT>, smem, done);
            if(rc != B200WMMA_OK)
                return rc;
            const PairParams p{q.c, q.d, q.m, q.n, q.k, q.ldc, q.ldd, q.alpha, q.beta, 16u, q.c ? P_STAGES_C : P_STAGES, q.c ? BOXES_C : BOXES,
                               q.status};
            const uint32_t   pairs = uint32_t(tiles < uint64_t(sms / 2) ? tiles : uint64_t(sms / 2));
            return cudaToStatus(launchOverlapped(mxGemmPairKernel<KIND, OutT>, dim3(2u * pairs), dim3(P_THREADS), smem,
                                                 stream, mapA, mapB, mapScaleA, mapScaleB, mapC, mapD, p));
        }

        template <ScaleKind KIND, typename OutT>
        int launchThin(Operands const& o, Params const& q, int sms, cudaStream_t stream)
        {
            constexpr uint32_t GROUPS = slotGroups<KIND>();
            const uint32_t     groups = mxGroups(KIND == ScaleKind::E4M3_16, q.k);
            const bool         thinA  = q.m <= q.n; // the thin operand is A
            ThinParams         p{};
            p.c      = q.c;
            p.d      = q.d;
            p.rows   = thinA ? q.n : q.m;
            p.thin   = thinA ? q.m : q.n;
            p.k      = q.k;
            p.cRow   = thinA ? 1u : q.ldc;
            p.cThin  = thinA ? q.ldc : 1u;
            p.dRow   = thinA ? 1u : q.ldd;
            p.dThin  = thinA ? q.ldd : 1u;
            p.alpha  = q.alpha;
            p.beta   = q.beta;
            p.status = q.status;
            p.r      = thinA ? o.b : o.a;
            p.ldr    = thinA ? o.ldb : o.lda;
            p.nq     = (p.thin + 15u) / 16u * 16u;
            const uint32_t slots = (q.k + SLOT_K - 1u) / SLOT_K;
            const uint32_t tiles = mxRowTiles(p.rows);
            // K is split until the blocks fill the device: twice over for up to 32 thin rows (1 x 8192 x
            // 8192 MXF4: 8.9 us with 4 parts, 10.3 with 2, 11.5 with 1, 11.9 with 8), once for more, whose
            // sums cost more to exchange (96 x 4096 x 4096 MXF4 f32: 7.1 us with 4 parts, 9.7 with 8; the
            // border is coarse: 64 x 16384 x 4096 NVF4 takes 12.0 with 1 part and 10.9 with 2).
            const uint32_t resident = p.nq <= 32u ? 2u : 1u;
            p.parts                 = 8;
            while(p.parts > 1u && (uint64_t(tiles) * p.parts > resident * uint32_t(sms) || slots < 2u * p.parts))
                p.parts /= 2u;
            p.slotBytes = CODE_BYTES + p.nq * 128u + GROUPS * MX_TILE_BYTES * 2u;
            // a block leaves room for another on its SM: of this kernel or of the next one
            const uint32_t room  = 112u * 1024u - uint32_t(sizeof(ThinControl)) - 1024u;
            const uint32_t mine  = (slots + p.parts - 1u) / p.parts;
            p.stages             = room / p.slotBytes;
            p.stages             = p.stages > MAX_STAGES ? MAX_STAGES : p.stages;
            p.stages             = p.stages > mine ? mine : p.stages;
            // the sums take the ring's place
            while(p.stages * p.slotBytes < p.nq * ROW_TILE * 4u)
                ++p.stages;
            const uint32_t cols = (p.nq + 31u) / 32u * 32u + 2u * 4u * GROUPS * 2u;
            p.tmemCols          = 32;
            while(p.tmemCols < cols)
                p.tmemCols *= 2;
            CUtensorMap mapR, mapQ, mapScaleR, mapScaleQ;
            int         rc = codeMap(&mapR, thinA ? o.b : o.a, p.rows, p.k, thinA ? o.ldb : o.lda, ROW_TILE);
            if(rc == B200WMMA_OK)
                rc = codeMap(&mapQ, thinA ? o.a : o.b, p.thin, p.k, thinA ? o.lda : o.ldb, p.nq);
            if(rc == B200WMMA_OK)
                rc = scaleMap(&mapScaleR, thinA ? o.bScales : o.aScales, p.rows, groups, GROUPS, 1);
            if(rc == B200WMMA_OK)
                rc = scaleMap(&mapScaleQ, thinA ? o.aScales : o.bScales, p.thin, groups, GROUPS, 1);
            if(rc != B200WMMA_OK)
                return rc;
            // A block takes at least the share of its SM's shared memory that it takes of the 512 columns, so
            // that an SM is not given more blocks than it has columns for, which would wait in
            // tcgen05.alloc while other SMs have room.  (That such a wait ends does not rest on this:
            // see the kernel.)
            constexpr uint32_t SM_SMEM = 228u * 1024u, BLOCK_SMEM = 1024u; // of an SM; on top of each block's own
            const uint32_t     share   = p.tmemCols * (SM_SMEM / 512u) - BLOCK_SMEM;
            uint32_t           smem    = 1024u + p.stages * p.slotBytes + uint32_t(sizeof(ThinControl));
            smem                       = smem < share ? share : smem;
            static uint32_t done[64] = {};
            rc = optInSharedMemory(mxGemmThinKernel<KIND, OutT>, smem, done);
            if(rc != B200WMMA_OK)
                return rc;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim            = dim3(tiles * p.parts);
            cfg.blockDim           = dim3(NUM_THREADS);
            cfg.dynamicSmemBytes   = smem;
            cfg.stream             = stream;
            cudaLaunchAttribute attr[2];
            attr[0].id               = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = p.parts;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            attr[1].id               = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[1].val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs    = attr;
            cfg.numAttrs = launchOverlapEnabled() ? 2 : 1;
            return cudaToStatus(cudaLaunchKernelEx(&cfg, mxGemmThinKernel<KIND, OutT>, mapR, mapQ, mapScaleR, mapScaleQ, p));
        }

        template <ScaleKind KIND, typename OutT>
        int launch(Operands const& o, Params const& p, cudaStream_t stream)
        {
            const int sms = smCount();
            if(sms < 2)
                return B200WMMA_ERR_CUDA;
            const uint32_t thin = p.m < p.n ? p.m : p.n;
            // (MXF4, 96 x 4096 x 4096 f32: 7.2 us thin, 12.1 in pairs; 128 x 8192 x 8192 bf16: 13.6 and 16.5)
            return thin <= THIN_ROWS ? launchThin<KIND, OutT>(o, p, sms, stream) : launchPairs<KIND, OutT>(o, p, sms, stream);
        }

        template <typename OutT>
        int launchFormat(int fmt, Operands const& o, Params const& p, cudaStream_t stream)
        {
            return fmt == B200WMMA_NVF4 ? launch<ScaleKind::E4M3_16, OutT>(o, p, stream)
                                        : launch<ScaleKind::E8M0_32, OutT>(o, p, stream);
        }
    } // namespace
} // namespace b200wmma

using namespace b200wmma;

extern "C" int b200wmma_mx_gemm(int fmt, int out_dtype, uint32_t m, uint32_t n, uint32_t k,
                                const void* a, const void* a_scales, const void* b,
                                const void* b_scales, const void* c, void* d, uint64_t lda,
                                uint64_t ldb, uint32_t ldc, uint32_t ldd, double alpha,
                                double beta, void* stream)
{
    if(!a || !a_scales || !b || !b_scales || !d || m == 0 || n == 0 || k == 0 || ldd < n
       || lda < mxPitch(k) || ldb < mxPitch(k) || (beta != 0.0 && (!c || ldc < n)))
        return B200WMMA_ERR_INVALID_ARG;
    if(!mxFormat(fmt)
       || (out_dtype != B200WMMA_F16 && out_dtype != B200WMMA_BF16 && out_dtype != B200WMMA_F32))
        return B200WMMA_ERR_UNSUPPORTED;
    const size_t size    = dtypeSize(out_dtype);
    auto         aligned = [](void const* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    if(!aligned(a) || !aligned(a_scales) || !aligned(b) || !aligned(b_scales) || !aligned(d)
       || lda % 16 || ldb % 16 || (ldd * size) % 16 || (beta != 0.0 && (!aligned(c) || (ldc * size) % 16)))
        return B200WMMA_ERR_ALIGNMENT;
    // coordinates of a TMA box are signed 32-bit numbers; a row of codes is k / 2 bytes
    if(m > 0x7fffff00u || n > 0x7fffff00u || k > 0x7fffff00u || lda >= (1ull << 40) || ldb >= (1ull << 40))
        return B200WMMA_ERR_TOO_LARGE;
    uint32_t* status = deviceStatusWord();
    if(!status)
        return B200WMMA_ERR_CUDA;
    const Operands     o{a, a_scales, b, b_scales, lda, ldb};
    const Params       p{beta != 0.0 ? c : nullptr, d, m, n, k, ldc, ldd, float(alpha), float(beta), status};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch(out_dtype)
    {
    case B200WMMA_F16:
        return launchFormat<__half>(fmt, o, p, s);
    case B200WMMA_BF16:
        return launchFormat<__nv_bfloat16>(fmt, o, p, s);
    }
    return launchFormat<float>(fmt, o, p, s);
}
