// Shared host/device helpers of the library: status word, tensor-map encoding
// through the driver entry point, argument checks.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200q {

// Device-side status word: 0 = ok; a bounded wait that ran out stores where it gave
// up (see ptx::mbar_wait).  One word per device, defined in common.cu; kernels get
// its device address as a parameter.
uint32_t* status_ptr();   // device address for the current device (nullptr on error)

// cuTensorMapEncodeTiled obtained with cudaGetDriverEntryPoint, so the library has no
// link-time dependency on libcuda.
CUresult encode_tiled(CUtensorMap* map, CUtensorMapDataType dtype, uint32_t rank, const void* gaddr,
                      const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                      CUtensorMapSwizzle swizzle);

// 2-D row-major byte matrix [rows, row_bytes] with a (box_rows x box_bytes) box.
// Out-of-range box elements are read as zero.
bool make_tmap_2d_u8(CUtensorMap* map, const void* gaddr, uint64_t rows, uint64_t row_bytes,
                     uint64_t row_stride_bytes, uint32_t box_rows, uint32_t box_bytes,
                     CUtensorMapSwizzle swizzle);

int num_sms();

// Tensor memory and clusters.  A CTA that allocates tensor memory waits, without a limit, for CTAs of the same SM to free theirs.  In a
// cluster those may in turn wait for a peer of their own that is short of tensor memory on another SM: a circle, from any two clustered
// kernels on two streams.  So whichever of them share an SM must fit its 512 columns together, and shared memory sees to it: a
// CTA that takes all columns asks for at least kWholeTmemSmem bytes, one that takes half of them for at least kHalfTmemSmem.  Two
// halves fit an SM (228 KB, 1 KB of each CTA kept by the system); three halves, a half and a whole, or two wholes do not.
// (CTAs without a cluster end by themselves; waiting for one closes no circle.)
constexpr int kSmSmem = 228 * 1024, kSystemSmem = 1024;
constexpr int kWholeTmemSmem = 120 * 1024, kHalfTmemSmem = 108 * 1024, kHalfTmemSmemMost = 113 * 1024;
static_assert(2 * (kHalfTmemSmemMost + kSystemSmem) <= kSmSmem && 3 * (kHalfTmemSmem + kSystemSmem) > kSmSmem &&
              kHalfTmemSmem + kWholeTmemSmem + 2 * kSystemSmem > kSmSmem && 2 * (kWholeTmemSmem + kSystemSmem) > kSmSmem, "who shares an SM");

// Tile order of the persistent CTA-pair GEMMs: `group` tile rows walk the N tiles together, so the A rows of a group
// stay in L2 while B streams past them once per group.  Measured (8192^3 FP8 and NVFP4, the MLP shapes): the best
// group is the largest power of two whose A rows fit in about 60 MB of the 126 MB L2.
inline int choose_tile_group(int tiles_m, size_t rows_per_tile, size_t row_bytes)
{
    const size_t budget = 60u << 20;
    int g = 1;
    while (g < tiles_m && g * 2 <= 64 && static_cast<size_t>(g * 2) * rows_per_tile * row_bytes <= budget) g *= 2;
    return g;
}

__host__ __device__ inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi)
{
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

}  // namespace b200q
