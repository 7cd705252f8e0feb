// MXFP4 block-scaled GEMM for sm_100a: host entry points and the kernel for few rows of A.
//   C[M,N] (bf16) = (A .* 2^(sfa - 127)) * (B .* 2^(sfb - 127))^T
// A[M,K/2], B[N,K/2]: two E2M1 per byte, low nibble = lower K; one UE8M0 scale (2^(byte - 127), 255 = NaN) per 32
// consecutive K; fp32 accumulate, one round-to-nearest-even cast to bf16 (data format:
// op/test/arch_primitives/ptx_mma_fp4.cu:49-53,120-130; scale decoder op/test/arch_primitives/ptx_mma_fp6.cu:344-351).
//
// Many rows: the CTA-pair block-scaled kernel of gemm_nvfp4_2cta.cu instantiated for this format.
// Few rows (decode), or few tiles: the product is bound by the bytes of B (K/2 + K/32 per row), so the kernel below is built to
// stream them.  It computes the transposed tile D[n, m] = sum_k B[n,k] A[m,k]: 128 rows of B fill the 128 lanes of the
// tensor-core tile, and the rows of A (16 to 128) are its narrow side, so no MMA work is spent on rows that are not there.
// K is split over the CTAs of a cluster so that even a square projection puts about two CTAs on every SM; the partial
// sums meet in shared memory (each CTA adds its share of the tile over the cluster in rank order, so the result does
// not depend on timing).
#include "common.cuh"
#include "ptx.cuh"
#include "../../include/b200q.h"

namespace b200q {

// gemm_nvfp4_2cta.cu
int gemm_block_scaled_pair(int fmt, const void* Aq, const void* SFA_blocked, const void* Bq, const void* SFB_blocked,
                           void* C, int M, int N, int K, float alpha, int bn, void* stream);

namespace mxfp4 {

constexpr int kBN = 128;                       // rows of B per tile (TMEM lanes)
constexpr int kSlabBytes = 128;                // per operand row and stage: 256 E2M1
constexpr int kSlabElems = 256;
constexpr int kSfBytes = 1024;                 // two 512-byte scale blocks (128 rows x 128 K each) per operand and stage
constexpr int kThreads = 192;                  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue (one per TMEM lane quadrant)
constexpr int kMaxStages = 8;
constexpr uint32_t kTmemCols = 256;            // accumulator (up to 128) + scales (8 + 8); two CTAs fit an SM

struct Params {
    int M, N, slabs, ksteps;                   // K slabs of 256 and MMAs of 64 along K
    int mt, stages, stage_bytes;               // rows of A per tile, depth of the load ring
    __nv_bfloat16* C;
    uint32_t* status;
};

__global__ void __launch_bounds__(kThreads)
gemm_mxfp4_few_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                           const __grid_constant__ CUtensorMap tmSFW, const __grid_constant__ CUtensorMap tmSFX, const Params p)
{
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bar_base = smem_base + p.stages * p.stage_bytes;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kMaxStages + s); };
    const uint32_t done_bar = bar_base + 8u * (2 * kMaxStages);
    const uint32_t tmem_slot = done_bar + 8u;
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - ptx::smem_u32(smem_raw)));
    float* partial = reinterpret_cast<float*>(smem_raw + (smem_base - ptx::smem_u32(smem_raw)));   // [mt][128], over the drained ring

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int splits = gridDim.x, split = blockIdx.x;            // the cluster spans x
    const int n0 = blockIdx.y * kBN, m0 = blockIdx.z * p.mt;
    const int slab0 = static_cast<int>(static_cast<long long>(p.slabs) * split / splits);
    const int slab1 = static_cast<int>(static_cast<long long>(p.slabs) * (split + 1) / splits);
    const uint32_t x_bytes = static_cast<uint32_t>(p.mt) * kSlabBytes;
    const uint32_t load_bytes = kBN * kSlabBytes + x_bytes + 2 * kSfBytes;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) { ptx::mbar_init(full_bar(s), 1); ptx::mbar_init(empty_bar(s), 1); }
        ptx::mbar_init(done_bar, 1);
        ptx::fence_mbar_init();
    }
    if (warp == 1) { ptx::tmem_alloc(tmem_slot, kTmemCols); ptx::tmem_relinquish(); }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot_ptr;

    if (warp == 0) {
        if (ptx::elect_one()) {
            ptx::tma_prefetch_desc(&tmW); ptx::tma_prefetch_desc(&tmX);
            ptx::tma_prefetch_desc(&tmSFW); ptx::tma_prefetch_desc(&tmSFX);
            // The launch does not wait for the kernel before this one (normally the quantiser of A): what comes before this line runs
            // beside it.  B waits too, since that kernel may have written it; bringing B into L2 meanwhile (prefetches are hints) did
            // not pay: 11.7 us for quantiser and product of 1 x 8192 x 8192 with it, 10.5 us without.
            ptx::pdl_wait();
            int stage = 0; uint32_t phase = 0; bool ok = true;
            for (int sl = slab0; sl < slab1 && ok; ++sl) {
                if (!ptx::mbar_wait(empty_bar(stage), phase ^ 1u, p.status, 1)) { ok = false; break; }
                const uint32_t sw = smem_base + stage * p.stage_bytes;
                const uint32_t sx = sw + kBN * kSlabBytes, ssfw = sx + x_bytes, ssfx = ssfw + kSfBytes;
                ptx::mbar_arrive_expect_tx(full_bar(stage), load_bytes);
                ptx::tma_load_2d(sw, &tmW, full_bar(stage), sl * kSlabBytes, n0);
                ptx::tma_load_2d(sx, &tmX, full_bar(stage), sl * kSlabBytes, m0);
                // the blocked scales as [row block][rows of 256 bytes]: a slab is two blocks = four such rows
                ptx::tma_load_3d(ssfw, &tmSFW, full_bar(stage), 0, 4 * sl, n0 / 128);
                ptx::tma_load_3d(ssfx, &tmSFX, full_bar(stage), 0, 4 * sl, m0 / 128);
                if (++stage == p.stages) { stage = 0; phase ^= 1u; }
            }
            if (!ok) __nanosleep(200000);                        // let loads in flight land before the CTA leaves
        }
    } else if (warp == 1) {
        ptx::pdl_wait();                                         // (the kernel before this one does not count against the waits' limit)
        if (ptx::elect_one()) {
            const uint32_t idesc = ptx::umma_idesc_block_scaled(1, 1, kBN, p.mt, 0, 0, 1);
            const uint32_t tsfw = tmem_base + 128, tsfx = tsfw + 8;
            int stage = 0; uint32_t phase = 0; bool ok = true;
            for (int sl = slab0; sl < slab1; ++sl) {
                if (!ptx::mbar_wait(full_bar(stage), phase, p.status, 3)) { ok = false; break; }
                ptx::tcgen05_fence_after_sync();
                const uint32_t sw = smem_base + stage * p.stage_bytes;
                const uint32_t sx = sw + kBN * kSlabBytes, ssfw = sx + x_bytes, ssfx = ssfw + kSfBytes;
                const uint64_t dw = ptx::smem_desc_sw128_kmajor(sw), dx = ptx::smem_desc_sw128_kmajor(sx);
                const uint64_t dsfw = ptx::smem_desc_noswizzle_kmajor(ssfw, 16, 128), dsfx = ptx::smem_desc_noswizzle_kmajor(ssfx, 16, 128);
                const int ksteps = min(4, p.ksteps - 4 * sl);
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    if (ks >= ksteps) break;
                    const int h = ks >> 1;
                    if ((ks & 1) == 0) {
                        ptx::tmem_cp_32x128b_warpx4(tsfw + 4 * h, dsfw + 32u * h);
                        ptx::tmem_cp_32x128b_warpx4(tsfx + 4 * h, dsfx + 32u * h);
                    }
                    const uint32_t id = idesc | (static_cast<uint32_t>(2 * (ks & 1)) << 4) | (static_cast<uint32_t>(2 * (ks & 1)) << 29);
                    ptx::umma_mxf4(tmem_base, dw + 2u * ks, dx + 2u * ks, id, tsfw + 4 * h, tsfx + 4 * h, sl > slab0 || ks > 0);
                }
                ptx::umma_commit(empty_bar(stage));
                if (++stage == p.stages) { stage = 0; phase ^= 1u; }
            }
            if (ok) ptx::umma_commit(done_bar);
            else __nanosleep(200000);
        }
    } else {
        // accumulator lane = row of B (output column), accumulator column = row of A (output row): for one output row a
        // warp stores 32 neighbouring columns
        ptx::pdl_wait();
        const int q = warp & 3;
        const int n = n0 + q * 32 + lane;
        const bool ok = ptx::mbar_wait(done_bar, 0, p.status, 4);
        if (ok) {
            ptx::tcgen05_fence_after_sync();
            for (int c = 0; c < p.mt; c += 16) {
                uint32_t r[16];
                ptx::tmem_ld_32x32b_x16(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + c, r);
                ptx::tmem_ld_wait();
                if (splits > 1) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) partial[(c + i) * kBN + q * 32 + lane] = __uint_as_float(r[i]);
                } else if (n < p.N) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (m0 + c + i < p.M) p.C[static_cast<size_t>(m0 + c + i) * p.N + n] = __float2bfloat16_rn(__uint_as_float(r[i]));
                }
            }
        }
    }
    ptx::tcgen05_fence_before_sync();
    if (splits > 1) {
        ptx::cluster_arrive();
        ptx::cluster_wait();
        // this CTA's share of the tile's rows, summed over the cluster in rank order
        const int quads = min(p.mt, p.M - m0) * (kBN / 4);
        for (int e = split * kThreads + threadIdx.x; e < quads; e += splits * kThreads) {
            const uint32_t at = smem_base + 16u * e;
            float4 v[8];
#pragma unroll
            for (int s = 0; s < 8; ++s) v[s] = s < splits ? ptx::ld_dsmem_f32x4(ptx::mapa(at, s)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float4 t = v[0];
#pragma unroll
            for (int s = 1; s < 8; ++s) { t.x += v[s].x; t.y += v[s].y; t.z += v[s].z; t.w += v[s].w; }
            const int m = m0 + e / (kBN / 4), n = n0 + e % (kBN / 4) * 4;
            __nv_bfloat16* to = p.C + static_cast<size_t>(m) * p.N + n;
            if (n + 4 <= p.N && (reinterpret_cast<uintptr_t>(to) & 7u) == 0) {
                *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(t.x, t.y), pack_bf16x2(t.z, t.w));
            } else {
                const float w[4] = {t.x, t.y, t.z, t.w};
                for (int i = 0; i < 4; ++i)
                    if (n + i < p.N) to[i] = __float2bfloat16_rn(w[i]);
            }
        }
        ptx::cluster_arrive();                 // a CTA's shared memory must outlive its peers' reads
        ptx::cluster_wait();
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, kTmemCols);
    }
}

int few_rows(const void* X, const void* SFX, const void* W, const void* SFW, void* C, int M, int N, int K, void* stream)
{
    const int sms = num_sms();
    if (sms <= 0) return cudaErrorInvalidDevice;
    Params p{};
    p.M = M; p.N = N; p.C = static_cast<__nv_bfloat16*>(C);
    p.slabs = (K + kSlabElems - 1) / kSlabElems; p.ksteps = (K + 63) / 64;
    p.mt = M >= 128 ? 128 : (M + 15) / 16 * 16;
    p.status = status_ptr();
    if (p.status == nullptr) return cudaErrorInvalidDevice;
    p.stage_bytes = (kBN * kSlabBytes + p.mt * kSlabBytes + 2 * kSfBytes + 1023) / 1024 * 1024;
    const int tiles_n = (N + kBN - 1) / kBN, tiles_m = (M + p.mt - 1) / p.mt;
    if (tiles_n > 65535 || tiles_m > 65535) return cudaErrorInvalidValue;
    // as many K splits as still give every CTA of two per SM at most one tile and every split four slabs
    int splits = 1;
    while (splits < 8 && static_cast<long long>(tiles_n) * tiles_m * splits * 2 <= 2LL * sms && p.slabs >= 4 * splits * 2) splits *= 2;
    const int per_split = (p.slabs + splits - 1) / splits;
    constexpr int kRingMost = 108 * 1024;
    static_assert(kRingMost + 1280 <= kHalfTmemSmemMost && kTmemCols == 256, "who shares an SM");
    const int budget = kRingMost / p.stage_bytes;
    p.stages = per_split < budget ? per_split : budget;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    if (p.stages < 1) p.stages = 1;
    // the ring doubles as the exchange buffer of the partial sums
    int ring = p.stages * p.stage_bytes;
    if (splits > 1 && ring < p.mt * kBN * 4) { p.stages = (p.mt * kBN * 4 + p.stage_bytes - 1) / p.stage_bytes; ring = p.stages * p.stage_bytes; }
    // enough that no more than two CTAs whose tensor memory fits become resident, of this kernel or of another clustered one (common.cuh)
    const int smem = ring + 1280 > kHalfTmemSmem ? ring + 1280 : kHalfTmemSmem;

    CUtensorMap tmW, tmX, tmSFW, tmSFX;
    const uint64_t row_bytes = static_cast<uint64_t>(K) / 2;
    if (!make_tmap_2d_u8(&tmW, W, N, row_bytes, row_bytes, kBN, kSlabBytes, CU_TENSOR_MAP_SWIZZLE_128B)) return cudaErrorInvalidValue;
    if (!make_tmap_2d_u8(&tmX, X, M, row_bytes, row_bytes, p.mt, kSlabBytes, CU_TENSOR_MAP_SWIZZLE_128B)) return cudaErrorInvalidValue;
    const uint64_t k_rows = static_cast<uint64_t>((K + 127) / 128) * 2;
    const uint64_t strides[2] = {256, k_rows * 256};
    const uint64_t dims_w[3] = {256, k_rows, static_cast<uint64_t>((N + 127) / 128)};
    const uint64_t dims_x[3] = {256, k_rows, static_cast<uint64_t>((M + 127) / 128)};
    const uint32_t box[3] = {256, 4, 1};
    if (encode_tiled(&tmSFW, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, SFW, dims_w, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    if (encode_tiled(&tmSFX, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, SFX, dims_x, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;

    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(gemm_mxfp4_few_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kHalfTmemSmemMost);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured[dev] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(splits, tiles_n, tiles_m); cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem; cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, gemm_mxfp4_few_rows_kernel, tmW, tmX, tmSFW, tmSFX, p);
}

}  // namespace mxfp4
}  // namespace b200q

extern "C" {

int b200q_gemm_mxfp4_blocked(const void* A, const void* SFA_blocked, const void* B, const void* SFB_blocked, void* C,
                             int M, int N, int K, void* stream)
{
    using namespace b200q;
    if (A == nullptr || SFA_blocked == nullptr || B == nullptr || SFB_blocked == nullptr || C == nullptr) return cudaErrorInvalidValue;
    if (M <= 0 || N <= 0 || K <= 0 || K % 32 != 0) return cudaErrorInvalidValue;
    if (!aligned16(A) || !aligned16(B) || !aligned16(SFA_blocked) || !aligned16(SFB_blocked)) return cudaErrorInvalidValue;
    const long long tiles_m = (M + 255) / 256, pairs = num_sms() / 2, tiles = tiles_m * ((N + 127) / 128);
    if (pairs <= 0) return cudaErrorInvalidDevice;
    // Up to 128 rows, and where the other kernel would have few tiles of a long K: this one splits K (256 x 1024: 7.0 us against 7.7
    // with K = 4096, 11.3 and 17.0 with 16384; 256 x 2560, 20 tiles: 9.2 and 7.9, 15.0 and 18.9; 600 x 1000 x 2048: 8.0 and 6.5).
    // Its grid has a row of clusters per 128 columns, which ends at 65535; the other kernel is persistent.
    constexpr int kMostN = 65535 * mxfp4::kBN;
    if ((M <= 128 && N <= kMostN) || (K >= 4096 && tiles <= (K >= 16384 ? 20 : 12)))
        return mxfp4::few_rows(A, SFA_blocked, B, SFB_blocked, C, M, N, K, stream);
    // Tiles of 128 columns where that leaves each CTA pair one at most (256 x 8192 x 8192: 13.0 us, 14.1 with 192, 16.3 with 256); else
    // the width whose last wave of CTA pairs wastes less, 192 where it fits the same number of waves (512 x 8192 x 8192: 22.0 us with
    // 192 columns, 16.5 with 256; 512 x 6568 x 15360: 22.0 and 25.2, 32.3 with 128).
    auto cost = [&](int bn) { return (tiles_m * ((N + bn - 1) / bn) + pairs - 1) / pairs * bn; };
    const int bn = tiles <= pairs ? 128 : cost(192) < cost(256) ? 192 : 256;
    return gemm_block_scaled_pair(2, A, SFA_blocked, B, SFB_blocked, C, M, N, K, 1.0f, bn, stream);
}

// Both MX formats share the scale layout: one UE8M0 byte per 32 K, 512-byte blocks of 128 rows x 128 K.
size_t b200q_gemm_mxfp4_workspace_bytes(int M, int N, int K) { return b200q_gemm_mxfp8_workspace_bytes(M, N, K); }

int b200q_gemm_mxfp4(const void* A, const void* SFA, const void* B, const void* SFB, void* C, int M, int N, int K,
                     void* workspace, void* stream)
{
    if (A == nullptr || B == nullptr || C == nullptr) return cudaErrorInvalidValue;
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return cudaErrorInvalidValue;
    const size_t a_bytes = b200q_mxfp8_sf_bytes(M, K);
    if (a_bytes == 0) return cudaErrorInvalidValue;
    uint8_t* wa = static_cast<uint8_t*>(workspace);
    uint8_t* wb = wa + a_bytes;
    int e = b200q_mxfp8_swizzle_sf(SFA, wa, M, K, stream);
    if (e != 0) return e;
    e = b200q_mxfp8_swizzle_sf(SFB, wb, N, K, stream);
    if (e != 0) return e;
    return b200q_gemm_mxfp4_blocked(A, wa, B, wb, C, M, N, K, stream);
}

}  // extern "C"
