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
#include <cuda.h>
#include <mutex>

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
        constexpr uint32_t EPI_THREADS = 128;
        constexpr uint32_t MAX_STAGES  = 8;

        struct Params
        {
            void const* c;
            void*       d;
            uint32_t    m, n, k, ldc, ldd;
            float       alpha, beta;
            uint32_t    nq, stages, slotBytes, tilesQ, tmemCols;
            uint32_t*   status;
        };

        struct Control
        {
            uint64_t   full[MAX_STAGES], empty[MAX_STAGES], accFull;
            AbortState abort;
            uint32_t   tmemBase;
        };

        template <ScaleKind KIND>
        constexpr uint32_t slotGroups() // scale tiles of 128 rows in a ring slot
        {
            return KIND == ScaleKind::E4M3_16 ? 4u : 2u;
        }

        // alpha and beta as everywhere in this library: a rounded product each, a rounded sum.
        template <typename OutT>
        __device__ inline OutT finish(float acc, Params const& p, OutT const* c)
        {
            float r = __fmul_rn(p.alpha, acc);
            if(c)
                r = __fadd_rn(r, __fmul_rn(p.beta, toFloat(*c)));
            return fromFloat<OutT>(r);
        }

        // One block, one tile: 128 rows of B (the MMA's M) by nq rows of A (its N).
        template <ScaleKind KIND, typename OutT>
        __global__ void __launch_bounds__(NUM_THREADS)
            mxGemmKernel(const __grid_constant__ CUtensorMap mapR,
                         const __grid_constant__ CUtensorMap mapQ,
                         const __grid_constant__ CUtensorMap mapScaleR,
                         const __grid_constant__ CUtensorMap mapScaleQ, const Params p)
        {
            constexpr uint32_t GROUPS = slotGroups<KIND>();
            extern __shared__ uint8_t smemRaw[];
            uint8_t* ring = smemRaw + ((1024u - (smem_addr(smemRaw) & 1023u)) & 1023u);
            Control* ctl  = reinterpret_cast<Control*>(ring + p.stages * p.slotBytes);

            const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
            const uint32_t tileR = blockIdx.x / p.tilesQ, tileQ = blockIdx.x % p.tilesQ;
            const uint32_t numSlots = (p.k + SLOT_K - 1) / SLOT_K;
            const uint32_t tilesOfQ = (p.nq + 127u) / 128u; // scale row tiles of this block's A
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
                    for(uint32_t it = 0; it < numSlots; ++it)
                    {
                        const uint32_t s = it % p.stages, ph = (it / p.stages) & 1u;
                        if(!mbar_wait(&ctl->empty[s], ph ^ 1u, &ctl->abort, WAIT_STAGE_EMPTY))
                            break;
                        uint8_t* slot   = ring + s * p.slotBytes;
                        uint8_t* scales = slot + CODE_BYTES + qBytes;
                        mbar_expect_tx(&ctl->full[s], p.slotBytes);
                        tma_load_2d(slot, &mapR, &ctl->full[s], int32_t(it * 128u), int32_t(tileR * ROW_TILE));
                        tma_load_2d(slot + CODE_BYTES, &mapQ, &ctl->full[s], int32_t(it * 128u),
                                    int32_t(tileQ * p.nq));
                        tma_load_3d(scales, &mapScaleR, &ctl->full[s], 0, int32_t(it * GROUPS), int32_t(tileR));
                        tma_load_3d(scales + GROUPS * MX_TILE_BYTES, &mapScaleQ, &ctl->full[s], 0,
                                    int32_t(it * GROUPS), int32_t(tileQ * p.nq / 128u));
                    }
                }
            }
            else if(warp == 1)
            {
                if(elect_one())
                {
                    // accumulator, then the scales of two ring slots in turn
                    const uint32_t scaleCols = 4u * GROUPS * (1u + tilesOfQ);
                    const uint32_t scale0    = tmem + (p.nq + 31u) / 32u * 32u;
                    bool           ok        = true;
                    for(uint32_t it = 0; it < numSlots; ++it)
                    {
                        const uint32_t s = it % p.stages, ph = (it / p.stages) & 1u;
                        if(!mbar_wait(&ctl->full[s], ph, &ctl->abort, WAIT_STAGE_FULL))
                        {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                        const uint32_t rAddr = smem_addr(ring + s * p.slotBytes);
                        const uint32_t qAddr = rAddr + CODE_BYTES, sAddr = qAddr + qBytes;
                        const uint32_t scaleR = scale0 + (it & 1u) * scaleCols;
                        const uint32_t scaleQ = scaleR + 4u * GROUPS;
                        const uint32_t left   = p.k - it * SLOT_K;
                        const uint32_t steps  = left >= SLOT_K ? SLOT_K / MMA_K : (left + MMA_K - 1) / MMA_K;
                        for(uint32_t g = 0; g < GROUPS; ++g)
                        {
                            tmem_copy_scales(scaleR + 4u * g, smem_desc_scales(sAddr + g * MX_TILE_BYTES));
                            for(uint32_t t = 0; t < tilesOfQ; ++t)
                                tmem_copy_scales(scaleQ + 4u * (g * tilesOfQ + t),
                                                 smem_desc_scales(sAddr + (GROUPS * (1u + t) + g) * MX_TILE_BYTES));
                        }
                        for(uint32_t ks = 0; ks < steps; ++ks)
                        {
                            // MXF4 takes a tile's four scales in two steps, NVF4 in one
                            const uint32_t g  = KIND == ScaleKind::E4M3_16 ? ks : ks / 2u;
                            const uint32_t id = KIND == ScaleKind::E4M3_16 ? 0u : (ks & 1u) * 2u;
                            mma_scaled<KIND>(tmem, smem_desc_kmajor_sw128(rAddr + ks * 32u),
                                             smem_desc_kmajor_sw128(qAddr + ks * 32u),
                                             make_instr_desc_scaled(KIND, ROW_TILE, p.nq, id),
                                             scaleR + 4u * g, scaleQ + 4u * g * tilesOfQ,
                                             (it > 0u || ks > 0u) ? 1u : 0u);
                        }
                        mma_commit(&ctl->empty[s]);
                    }
                    if(ok)
                        mma_commit(&ctl->accFull);
                }
            }
            else
            {
                // lanes hold rows of B (columns of D), registers rows of A (rows of D)
                const uint32_t quad = warp % 4;
                const uint32_t col  = tileR * ROW_TILE + quad * 32u + lane;
                const bool     ready = mbar_wait(&ctl->accFull, 0, &ctl->abort, WAIT_ACC_FULL);
                if(named_barrier_all(1, EPI_THREADS, ready))
                {
                    tc_fence_after_sync();
                    for(uint32_t j0 = 0; j0 < p.nq; j0 += 16u)
                    {
                        uint32_t raw[16];
                        tmem_load_32x32b_x16(tmem + ((quad * 32u) << 16) + j0, raw);
                        tmem_load_wait();
#pragma unroll
                        for(uint32_t j = 0; j < 16u; ++j)
                        {
                            const uint64_t row = uint64_t(tileQ) * p.nq + j0 + j;
                            if(row < p.m && col < p.n)
                            {
                                OutT const* c = p.c ? static_cast<OutT const*>(p.c) + row * p.ldc + col : nullptr;
                                static_cast<OutT*>(p.d)[row * p.ldd + col]
                                    = finish<OutT>(__uint_as_float(raw[j]), p, c);
                            }
                        }
                    }
                    tc_fence_before_sync();
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

        template <typename KernelT>
        int optInSharedMemory(KernelT kernel, uint32_t bytes, uint32_t (&done)[64])
        {
            static std::mutex           attrMutex;
            std::lock_guard<std::mutex> lock(attrMutex);
            int                         dev = 0;
            B200WMMA_CUDA_TRY(cudaGetDevice(&dev));
            if(dev < 0 || dev >= 64 || done[dev] < bytes)
            {
                B200WMMA_CUDA_TRY(cudaFuncSetAttribute(
                    kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
                if(dev >= 0 && dev < 64)
                    done[dev] = bytes;
            }
            return B200WMMA_OK;
        }

        struct Operands
        {
            void const *a, *aScales, *b, *bScales;
            uint64_t    lda, ldb;
        };

        template <ScaleKind KIND, typename OutT>
        int launch(Operands const& o, Params p, cudaStream_t stream)
        {
            constexpr uint32_t GROUPS = slotGroups<KIND>();
            const uint32_t     groups = mxGroups(KIND == ScaleKind::E4M3_16, p.k);
            p.nq                      = p.m > 128u ? 256u : p.m > 64u ? 128u : (p.m + 15u) / 16u * 16u;
            const uint32_t tilesOfQ   = (p.nq + 127u) / 128u;
            p.slotBytes               = CODE_BYTES + p.nq * 128u + GROUPS * MX_TILE_BYTES * (1u + tilesOfQ);
            p.stages                  = 4;
            p.tilesQ                  = uint32_t((uint64_t(p.m) + p.nq - 1) / p.nq);
            const uint32_t cols       = (p.nq + 31u) / 32u * 32u + 2u * 4u * GROUPS * (1u + tilesOfQ);
            p.tmemCols                = 32;
            while(p.tmemCols < cols)
                p.tmemCols *= 2;
            const uint64_t blocks = uint64_t(mxRowTiles(p.n)) * p.tilesQ;
            if(blocks > 0x7fffffffull)
                return B200WMMA_ERR_TOO_LARGE;
            CUtensorMap mapR, mapQ, mapScaleR, mapScaleQ;
            int         rc = codeMap(&mapR, o.b, p.n, p.k, o.ldb, ROW_TILE);
            if(rc == B200WMMA_OK)
                rc = codeMap(&mapQ, o.a, p.m, p.k, o.lda, p.nq);
            if(rc == B200WMMA_OK)
                rc = scaleMap(&mapScaleR, o.bScales, p.n, groups, GROUPS, 1);
            if(rc == B200WMMA_OK)
                rc = scaleMap(&mapScaleQ, o.aScales, p.m, groups, GROUPS, tilesOfQ);
            if(rc != B200WMMA_OK)
                return rc;
            const uint32_t  smem = 1024u + p.stages * p.slotBytes + uint32_t(sizeof(Control));
            static uint32_t done[64] = {};
            rc = optInSharedMemory(mxGemmKernel<KIND, OutT>, smem, done);
            if(rc != B200WMMA_OK)
                return rc;
            return cudaToStatus(launchOverlapped(mxGemmKernel<KIND, OutT>, dim3(uint32_t(blocks)),
                                                 dim3(NUM_THREADS), smem, stream, mapR, mapQ, mapScaleR,
                                                 mapScaleQ, p));
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
    const Params       p{beta != 0.0 ? c : nullptr, d, m, n, k, ldc, ldd, float(alpha), float(beta), 0, 0, 0, 0, 0, status};
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
