// Arguments of the paged attention's kernels, and what they share: the rows nobody owns, the log of the sum, the kernel that joins
// the parts of a block whose keys were split over CTAs.
#pragma once
#include "paged_common.cuh"
#include "ptx.cuh"

namespace b200q {
namespace paged {

struct Args {
    Shape s;
    const __nv_bfloat16* q;              // row (token, head) at token * q_stride + head * q_head elements
    long long q_stride, q_head;
    const void *k_cache, *v_cache;
    const float *k_scale, *v_scale;
    __nv_bfloat16* out;                  // [tokens, heads, D]
    float* lse;                          // [tokens, heads] or null
    float scale_log2;                    // softmax scale * log2(e)
    int max_q;                           // the caller's bound of the chunk lengths
    int block_limit;                     // ... in row blocks (only how the work is counted depends on it)
    int block_most;                      // bound of the call's blocks: row blocks of all sequences, times kv heads
    int zero_rest;                       // rows of no sequence: write zeros (else leave them)
    Open* open;                          // [CTAs]
    float* part;                         // [2 * CTAs][rows * D outputs, then rows x (max, sum)]
    uint32_t* status;
};

int attn_split(const Args& a, int head_dim, bool fp8, cudaStream_t stream);
int attn_chunk(const Args& a, int head_dim, bool fp8, cudaStream_t stream);
size_t attn_chunk_part_bytes(int head_dim);
int attn_split_ctas();                       // the most CTAs a launch uses
size_t attn_split_part_bytes(int head_dim);  // the most its parts take

// The most row blocks of a call, over all sequences and kv heads.
inline long long most_blocks(const Args& a, int rm)
{
    const long long each = (static_cast<long long>(a.max_q) * a.s.group + rm - 1) / rm;
    const long long all = static_cast<long long>(a.s.tokens) * a.s.group / rm + a.s.seqs;
    return (a.s.seqs * each < all ? a.s.seqs * each : all) * a.s.kv_heads;
}

// Whether the tiles of a call, however its arrays divide the rows and keys, can be counted in 32 bits.
inline bool tiles_fit(const Args& a, int rm, int kt)
{
    const double blocks = static_cast<double>(a.s.tokens) * a.s.group / rm + a.s.seqs;
    const double keys = static_cast<double>(a.s.max_pages) * (1 << a.s.page_shift);
    return blocks * a.s.kv_heads * (keys / kt + 2) < 2.0e9;
}

// natural log of sum_j e^(scale * q.k_j), from the maximum in units of log2 and the sum of 2^(x - max); -inf for no keys
__device__ __forceinline__ float lse_of(float m, float l)
{
    return l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// rows in front of the first and behind the last sequence
template <int D>
__device__ __forceinline__ void zero_rest(const Args& a)
{
    if (!a.zero_rest) return;
    const int lo = min(max(__ldg(a.s.cu_q), 0), a.s.tokens), hi = min(max(__ldg(a.s.cu_q + a.s.seqs), lo), a.s.tokens);
    if (lo == 0 && hi == a.s.tokens) return;
    const long long vecs = static_cast<long long>(a.s.heads) * (D / 8);
    const int rest = lo + a.s.tokens - hi;
    const long long block = static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x, blocks = static_cast<long long>(gridDim.x) * gridDim.y;
    for (long long i = block * blockDim.x + threadIdx.x; i < rest * vecs; i += blocks * blockDim.x) {
        int t = static_cast<int>(i / vecs);
        const long long e = i - t * vecs;
        if (t >= lo) t += hi - lo;
        reinterpret_cast<uint4*>(a.out)[t * vecs + e] = make_uint4(0, 0, 0, 0);
        if (a.lse != nullptr && e < a.s.heads) a.lse[static_cast<size_t>(t) * a.s.heads + e] = -INFINITY;
    }
}

// Joins the parts of every open block: CTA c's tail, then the leading parts of the CTAs up to the one that did the last
// tile, in that order (the result does not depend on timing).  One warp per row.
template <int D>
__global__ void __launch_bounds__(256)
combine_kernel(const Args a, int rows_per_block)
{
    constexpr int kPer = D / 32;
    zero_rest<D>(a);                           // (nothing else writes these rows)
    ptx::pdl_wait();
    const Open op = a.open[blockIdx.x];
    const int lane = threadIdx.x & 31;
    if (op.last < 0) return;
    for (int row = blockIdx.y * 8 + (threadIdx.x >> 5); row < op.rows; row += gridDim.y * 8) {
        const size_t slot_floats = static_cast<size_t>(rows_per_block) * (D + 2);
        const int c0 = blockIdx.x, parts = op.last - c0 + 1;
        auto part = [&](int i) { return a.part + static_cast<size_t>(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * slot_floats; };
        // a lane has the state of every 32nd part; 32 parts at a time, their outputs' loads are independent of one another
        float m = -INFINITY;
        for (int i = lane; i < parts; i += 32) m = ptx::max_nan(m, part(i)[rows_per_block * D + row * 2]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = ptx::max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, acc[kPer] = {};
        for (int i0 = 0; i0 < parts; i0 += 32) {
            float f = 0.0f;
            if (i0 + lane < parts) {
                const float2 st = *reinterpret_cast<const float2*>(part(i0 + lane) + rows_per_block * D + row * 2);
                f = ptx::ex2(st.x - base);
                l += st.y * f;
            }
            const int n = min(32, parts - i0);
#pragma unroll 8
            for (int i = 0; i < n; ++i) {
                const float* p = part(i0 + i) + row * D;
                const float fi = __shfl_sync(0xffffffffu, f, i);
                if constexpr (kPer == 4) {
                    const float4 v = *reinterpret_cast<const float4*>(p + lane * 4);
                    acc[0] += v.x * fi; acc[1] += v.y * fi; acc[2] += v.z * fi; acc[3] += v.w * fi;
                } else {
                    const float2 v = *reinterpret_cast<const float2*>(p + lane * 2);
                    acc[0] += v.x * fi; acc[1] += v.y * fi;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int r = op.r0 + row, t = a.s.token_of(r);
        const size_t to = static_cast<size_t>(op.token0 + t) * a.s.heads + op.h * a.s.group + r - t * a.s.group;
        const float inv = l == 0.0f ? 0.0f : __frcp_rn(l);
        if constexpr (kPer == 4)
            *reinterpret_cast<uint2*>(a.out + to * D + lane * 4) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
        else
            *reinterpret_cast<uint32_t*>(a.out + to * D + lane * 2) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
        if (a.lse != nullptr && lane == 0) a.lse[to] = lse_of(m, l);
    }
}

// The kernel may start while its predecessor runs (it waits for its results before it reads anything).
template <int D>
int launch_combine(const Args& a, int ctas, int rows_per_block, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg{};
    // eight rows a CTA, as many as a block has or the caller's bound of the chunk lengths allows
    const long long rows = static_cast<long long>(a.max_q) * a.s.group;
    const int most = rows < rows_per_block ? static_cast<int>(rows) : rows_per_block;
    cfg.gridDim = dim3(ctas, (most + 7) / 8); cfg.blockDim = dim3(256); cfg.stream = stream;
    // the split of shared memory and L1 that the kernel before it has: another one would have to wait for an idle SM
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(combine_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured[dev] = true;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, combine_kernel<D>, a, rows_per_block);
}

}  // namespace paged
}  // namespace b200q
