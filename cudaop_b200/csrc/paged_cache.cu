// Writing new tokens' keys and values into a paged cache (quantised on the way) and reading a batch of sequences back.
//
// Quantisation is the per-row rule of b200q_quant_rows_e4m3 with a row per (token, kv head):
//   s = max|x| / 448 (1 for a zero row, at least the smallest normal float),  byte = e4m3_rn(x * (1 / s)).
// A row that holds NaN or an infinity gets the scale NaN and zero bytes, so whatever reads it becomes NaN and no byte of
// the cache is ever NaN by itself.  Reading back is bf16_rn(float(byte) * s).
//
// Both are bound by HBM: 2 bytes read and 1 written per element (write), the reverse for reading back.  A thread moves 16
// bytes of bf16 per row and tensor, so a row of 128 is 16 lanes, a warp instruction covers whole 128- and 256-byte runs, and
// keys and values of the row are in flight together.
#include "common.cuh"
#include <cuda_fp8.h>
#include "../../include/b200q.h"

namespace b200q {
namespace paged {

constexpr int kThreads = 256;
constexpr int kTokens = 16;                  // tokens per CTA of the reading kernel

__device__ __forceinline__ float lo16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// 8 bf16 of a row of 8 * kLanes -> 8 E4M3 bytes and the row's scale
template <int kLanes>
__device__ __forceinline__ uint2 quantise8(uint4 u, float& scale)
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t m2 = 0;                         // magnitudes compare as integers, NaN > infinity > finite
#pragma unroll
    for (int k = 0; k < 4; ++k) m2 = __vmaxu2(m2, w[k] & 0x7FFF7FFFu);
    uint32_t mx = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m = __uint_as_float(mx << 16);
    const bool finite = mx < 0x7F80u;
    const float s = m > 0.0f ? fmaxf(__fdiv_rn(m, 448.0f), 1.17549435e-38f) : 1.0f;
    scale = finite ? s : __uint_as_float(0x7FC00000u);
    const float inv = __frcp_rn(s);
    uint32_t h[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        h[k] = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(lo16(w[k]), inv), __fmul_rn(hi16(w[k]), inv)), __NV_SATFINITE, __NV_E4M3);
    return finite ? make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16)) : make_uint2(0u, 0u);
}

__device__ __forceinline__ uint4 dequantise8(uint2 q, float s)
{
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t w = (k < 2 ? q.x : q.y) >> (16 * (k & 1));
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFFu), __NV_E4M3)));
        o[k] = pack_bf16x2(__fmul_rn(f.x, s), __fmul_rn(f.y, s));
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// k, v: rows of D bf16, (token, head) at token * stride + head * head_stride elements.  slots: token -> page * page_size +
// offset; a slot outside the cache is skipped.  A row is D / 8 lanes, and a thread has one piece of one row: the loads of the data and of
// the slot go out together (one decode step of 64 sequences, 8 heads: 8.1 us with 16 tokens a CTA in turns, 2.0 us so).
template <int D, bool FP8>
__global__ void __launch_bounds__(kThreads)
write_kernel(const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, long long k_stride, long long v_stride,
             long long k_head, long long v_head, const long long* __restrict__ slots, uint8_t* __restrict__ kc,
             uint8_t* __restrict__ vc, float* __restrict__ ks, float* __restrict__ vs, long long rows, int kv_heads,
             long long num_slots, int page_shift)
{
    constexpr int kLanes = D / 8;
    const int lane = threadIdx.x % kLanes;
    const long long i = static_cast<long long>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
    const bool in = i < rows;                // (no early return: the shuffles below need every lane)
    const long long t = in ? i / kv_heads : 0;
    const int h = in ? static_cast<int>(i - t * kv_heads) : 0;
    const long long slot = __ldg(slots + t);
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(k + t * k_stride + h * k_head) + lane);
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(v + t * v_stride + h * v_head) + lane);
    const bool on = in && slot >= 0 && slot < num_slots;
    const long long page = slot >> page_shift;
    const long long row = ((page * kv_heads + h) << page_shift) + (slot - (page << page_shift));
    if (FP8) {
        float sa, sb;
        const uint2 qa = quantise8<kLanes>(a, sa), qb = quantise8<kLanes>(b, sb);
        if (on) {
            *reinterpret_cast<uint2*>(kc + row * D + lane * 8) = qa;
            *reinterpret_cast<uint2*>(vc + row * D + lane * 8) = qb;
            if (lane == 0) { ks[row] = sa; vs[row] = sb; }
        }
    } else if (on) {
        reinterpret_cast<uint4*>(kc + row * D * 2)[lane] = a;
        reinterpret_cast<uint4*>(vc + row * D * 2)[lane] = b;
    }
}

// Row r of the output is token r - cu[b] of the sequence b with cu[b] <= r < cu[b + 1] (a start below zero counts as zero).  A token whose page number is outside
// the cache reads as zero.  Rows that belong to no sequence are left as they are, or zeroed (zero_rest).
template <int D, bool FP8>
__global__ void __launch_bounds__(kThreads)
read_kernel(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc, const float* __restrict__ ks, const float* __restrict__ vs,
            const int* __restrict__ table, const int* __restrict__ cu, __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v,
            int seqs, int total, int kv_heads, int max_pages, int num_pages, int page_shift, int zero_rest)
{
    constexpr int kLanes = D / 8;
    __shared__ long long row0[kTokens];      // cache row of (token, head 0); -1 = zero, -2 = leave
    const int t0 = blockIdx.x * kTokens;
    const int count = min(kTokens, total - t0);
    if (threadIdx.x < count) {
        const int r = t0 + threadIdx.x;
        int lo = 0, hi = seqs;               // first b with cu[b + 1] > r, or seqs
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (__ldg(cu + mid + 1) > r) hi = mid; else lo = mid + 1;
        }
        long long row = zero_rest ? -1 : -2;
        if (lo < seqs && r >= __ldg(cu + lo)) {
            // (0 <= j <= r whatever the array holds: r - cu[b] of a start near -2^31 would pass 32 bits and index in front of the table)
            const int j = r - max(__ldg(cu + lo), 0), col = j >> page_shift;
            const int page = col < max_pages ? __ldg(table + static_cast<size_t>(lo) * max_pages + col) : -1;
            row = page >= 0 && page < num_pages
                      ? ((static_cast<long long>(page) * kv_heads) << page_shift) + (j & ((1 << page_shift) - 1)) : -1;
        }
        row0[threadIdx.x] = row;
    }
    __syncthreads();
    const int lane = threadIdx.x % kLanes;
    const int items = count * kv_heads;
    constexpr int kStep = kThreads / kLanes, kAhead = 4;         // rows a thread has in flight
    for (int i0 = threadIdx.x / kLanes; i0 < items; i0 += kStep * kAhead) {
        long long row[kAhead];
        uint4 a[kAhead], b[kAhead];
        float sa[kAhead], sb[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + u * kStep;
            const int t = i / kv_heads, h = i - t * kv_heads;
            const long long base = i < items ? row0[t] : -2;
            row[u] = base < 0 ? base : base + (static_cast<long long>(h) << page_shift);
            a[u] = b[u] = make_uint4(0, 0, 0, 0);
            sa[u] = sb[u] = 1.0f;
            if (base >= 0) {
                if (FP8) {
                    const uint2 x = __ldg(reinterpret_cast<const uint2*>(kc + row[u] * D) + lane), y = __ldg(reinterpret_cast<const uint2*>(vc + row[u] * D) + lane);
                    a[u].x = x.x; a[u].y = x.y; b[u].x = y.x; b[u].y = y.y;
                    sa[u] = __ldg(ks + row[u]); sb[u] = __ldg(vs + row[u]);
                } else {
                    a[u] = __ldg(reinterpret_cast<const uint4*>(kc + row[u] * D * 2) + lane);
                    b[u] = __ldg(reinterpret_cast<const uint4*>(vc + row[u] * D * 2) + lane);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (row[u] == -2) continue;
            const int i = i0 + u * kStep;
            const size_t to = (static_cast<size_t>(t0) * kv_heads + i) * kLanes + lane;
            __stcs(reinterpret_cast<uint4*>(k) + to, FP8 ? dequantise8(make_uint2(a[u].x, a[u].y), sa[u]) : a[u]);
            __stcs(reinterpret_cast<uint4*>(v) + to, FP8 ? dequantise8(make_uint2(b[u].x, b[u].y), sb[u]) : b[u]);
        }
    }
}

// -1 for a page size that is not a power of two from 16 to 128
int page_shift_of(int page_size)
{
    for (int s = 4; s <= 7; ++s)
        if (page_size == 1 << s) return s;
    return -1;
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace paged
}  // namespace b200q

extern "C" {

int b200q_paged_cache_write(const void* k, const void* v, const long long* slots, void* k_cache, void* v_cache, float* k_scale,
                            float* v_scale, int tokens, int kv_heads, int head_dim, long long k_stride, long long v_stride,
                            long long k_head_stride, long long v_head_stride, int num_pages, int page_size, int fp8, void* stream)
{
    using namespace b200q;
    using namespace b200q::paged;
    if (k == nullptr || v == nullptr || slots == nullptr || k_cache == nullptr || v_cache == nullptr) return cudaErrorInvalidValue;
    if (fp8 && (k_scale == nullptr || v_scale == nullptr)) return cudaErrorInvalidValue;
    const int shift = page_shift_of(page_size);
    if (tokens <= 0 || kv_heads <= 0 || num_pages <= 0 || shift < 0 || (head_dim != 64 && head_dim != 128)) return cudaErrorInvalidValue;
    if (k_stride % 8 || v_stride % 8 || k_head_stride % 8 || v_head_stride % 8) return cudaErrorInvalidValue;
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned(slots, 8)) return cudaErrorInvalidValue;
    const long long num_slots = static_cast<long long>(num_pages) << shift;
    const long long rows = static_cast<long long>(tokens) * kv_heads;
    const long long grid = (rows * (head_dim / 8) + kThreads - 1) / kThreads;
    if (grid > 0x7FFFFFFFll) return cudaErrorInvalidValue;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto kernel) {
        kernel<<<static_cast<unsigned>(grid), kThreads, 0, st>>>(static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), k_stride, v_stride,
                                          k_head_stride, v_head_stride, slots, static_cast<uint8_t*>(k_cache),
                                          static_cast<uint8_t*>(v_cache), k_scale, v_scale, rows, kv_heads, num_slots, shift);
    };
    if (head_dim == 64) { if (fp8) run(write_kernel<64, true>); else run(write_kernel<64, false>); }
    else { if (fp8) run(write_kernel<128, true>); else run(write_kernel<128, false>); }
    return cudaGetLastError();
}

int b200q_paged_cache_read(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                           const int* page_table, const int* cu_kv, void* k, void* v, int seqs, int total, int kv_heads, int head_dim,
                           int max_pages, int num_pages, int page_size, int fp8, int zero_rest, void* stream)
{
    using namespace b200q;
    using namespace b200q::paged;
    if (k == nullptr || v == nullptr || cu_kv == nullptr || page_table == nullptr || k_cache == nullptr || v_cache == nullptr) return cudaErrorInvalidValue;
    if (fp8 && (k_scale == nullptr || v_scale == nullptr)) return cudaErrorInvalidValue;
    const int shift = page_shift_of(page_size);
    if (seqs <= 0 || total <= 0 || kv_heads <= 0 || max_pages <= 0 || num_pages <= 0 || shift < 0 || (head_dim != 64 && head_dim != 128))
        return cudaErrorInvalidValue;
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache)) return cudaErrorInvalidValue;
    const int grid = (total + kTokens - 1) / kTokens;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto run = [&](auto kernel) {
        kernel<<<grid, kThreads, 0, st>>>(static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), k_scale, v_scale,
                                          page_table, cu_kv, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), seqs, total,
                                          kv_heads, max_pages, num_pages, shift, zero_rest);
    };
    if (head_dim == 64) { if (fp8) run(read_kernel<64, true>); else run(read_kernel<64, false>); }
    else { if (fp8) run(read_kernel<128, true>); else run(read_kernel<128, false>); }
    return cudaGetLastError();
}

}  // extern "C"
