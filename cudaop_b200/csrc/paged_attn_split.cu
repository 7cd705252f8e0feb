// Attention of a chunk of new tokens over a paged cache, for few rows per kv head (decode, drafted tokens): the split-KV
// kernel and the kernel that joins its parts.
//
//   o[r,:] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x_j = scale * log2(e) * (q_r . k_j),  m = max_j x_j
// over the keys j that row r sees.  An E4M3 cache is never dequantised as such: the bytes become bf16 exactly (see e4m3x2 below),
// a key's scale multiplies the 32-bit product q.k and a value's scale multiplies p before it is rounded to bf16 for the second
// product.  That rounding of p (half a step, 2^-9 of a value's share) is the only one besides the output's; sums, maxima and
// accumulators are 32-bit.
//
// Bound by the bytes of the cache: with 16 rows the tensor work per byte is small, so the design is one pass over the keys at
// HBM rate.  A CTA is a producer warp that fills a ring of 64-key tiles by TMA (one box per page and tensor; the
// page table is read a tile ahead) and four consumer warps of 16 keys each: their softmax states are independent, so a tile needs no
// barrier but the ring's, and they meet once per block of rows.  m16n8k16 products with the rows as the 16 side; the contraction
// order over head_dim (and the order of output columns) is permuted so that every shared-memory read is a conflict-free
// 16 (or 8) byte load of consecutive elements.  The work is divided over the persistent grid by tiles (paged_common.cuh).
#include "paged_common.cuh"
#include "paged_attn.cuh"
#include "ptx.cuh"

namespace b200q {
namespace paged {
namespace split {

constexpr int kRows = 16, kTile = 64, kConsumers = 4, kThreads = 32 * (kConsumers + 1);

template <int D, bool FP8>
struct Cfg {
    static constexpr int kRowBytes = FP8 ? D : 2 * D;
    static constexpr int kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;       // inner extent of a box = swizzle span
    static constexpr int kHalves = kRowBytes / kBoxBytes;
    static constexpr int kHalfBytes = kTile * kBoxBytes;
    static constexpr int kTensorBytes = kTile * kRowBytes;
    static constexpr int kScaleBytes = FP8 ? kTile * 4 : 0;
    static constexpr int kStageBytes = (2 * kTensorBytes + 2 * kScaleBytes + 1023) / 1024 * 1024;
    static constexpr int kJoinBytes = kRows * D * 4;                          // one warp's accumulators
    static constexpr int kStages = (112 * 1024 - 2048 - kJoinBytes) / kStageBytes < 8 ? (112 * 1024 - 2048 - kJoinBytes) / kStageBytes : 8;
    static constexpr int kStateBytes = kConsumers * kRows * 8;                // running maximum and sum per warp and row
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kJoinBytes + kStateBytes + kStages * (8 + 16);
    static constexpr int kSteps = D / 16;                                     // k-steps of q.k
    static constexpr int kCols = D / 8;                                       // 8-column groups of the output
};

// Two E4M3 bytes, in bits 8..15 and 24..31 of x, as two bf16, exactly: sign and the seven exponent and mantissa bits go where
// bf16 has them, which reads as the value times 2^-120 (the exponent biases are 7 and 127; subnormals included), and one
// exact product puts that right.  NaN bytes do not occur (the write kernel stores none).
__device__ __forceinline__ uint32_t e4m3x2(uint32_t x)
{
    const uint32_t t = (x & 0x80008000u) | ((x >> 4) & 0x07F007F0u);
    __nv_bfloat162 v, c;
    *reinterpret_cast<uint32_t*>(&v) = t;
    *reinterpret_cast<uint32_t*>(&c) = 0x7B807B80u;                            // 2^120
    v = __hmul2(v, c);
    return *reinterpret_cast<uint32_t*>(&v);
}

// The row r of the block as its 16-bit elements in the order the products take them: k-step s gives thread c = lane % 4 the
// four consecutive elements that follow d0(s, c).
template <int D, bool FP8>
__device__ __forceinline__ int q_element(int s, int c)
{
    if (FP8) return D == 128 ? (2 * c + (s >> 2)) * 16 + 4 * (s & 3) : c * 16 + 4 * s;
    return (s >> 2) * 64 + (2 * c + ((s >> 1) & 1)) * 8 + 4 * (s & 1);
}

// bytes [16 * chunk, +16) of row `row` of a tile half whose rows are kBox bytes, 128- (64-) byte swizzle
template <int kBox>
__device__ __forceinline__ uint32_t swizzled(uint32_t base, int row, int byte)
{
    const uint32_t a = static_cast<uint32_t>(row) * kBox + byte;
    return base + (a ^ (kBox == 128 ? (a >> 3) & 0x70u : (a >> 3) & 0x30u));
}

template <int D, bool FP8>
__global__ void __launch_bounds__(kThreads, 2)
attn_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a)
{
    using C = Cfg<D, FP8>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    const uint32_t join = ring + C::kStages * C::kStageBytes;
    float* join_p = reinterpret_cast<float*>(smem_raw + (join - raw));
    float2* state_p = reinterpret_cast<float2*>(smem_raw + (join - raw) + C::kJoinBytes);         // [warp][row] (max, sum)
    unsigned long long* mask_p = reinterpret_cast<unsigned long long*>(smem_raw + (join - raw) + C::kJoinBytes + C::kStateBytes);
    const uint32_t bars = join + C::kJoinBytes + C::kStateBytes + 8 * C::kStages;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (C::kStages + s); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Shape& s = a.s;

    ptx::pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) { ptx::mbar_init(full_bar(i), 1); ptx::mbar_init(empty_bar(i), kConsumers); }
        ptx::fence_mbar_init();
    }
    zero_rest<D>(a);
    Cursor c = find_work(s, kRows, kTile, reinterpret_cast<long long*>(smem_raw + (ring - raw)), a.block_limit, blockIdx.x, gridDim.x);
    if (threadIdx.x == 0) a.open[blockIdx.x].last = -1;
    if (c.at == c.end) return;
    ptx::fence_proxy_async_smem();             // the ring held the prefix sums; the loads that follow are the async proxy's
    __syncthreads();
    Seq q = load_seq(s, c.b);

    if (warp == kConsumers) {
        // ------------------------------------------------------------------------------------------ producer
        const int box = min(kTile, 1 << s.page_shift);             // keys per box
        const int boxes = kTile / box;
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        while (c.at < c.end && ok) {
            const Range r = block_range(s, q, c.i, kRows, kTile);
            const int todo = static_cast<int>(min(static_cast<long long>(r.tiles - c.tile), c.end - c.at));
            const int* table = s.table + static_cast<size_t>(c.b) * s.max_pages;
            auto page_of = [&](int tile) {                          // lane < boxes: the page of its box of the tile, -1 for none
                const int key = tile * kTile + lane * box;
                const bool in = lane < boxes && key < r.hi && key + box > r.lo;
                const int p = in ? __ldg(table + (key >> s.page_shift)) : -1;
                return p >= 0 && p < s.num_pages ? p : -1;
            };
            int page = page_of(r.tile0 + c.tile);
            for (int t = 0; t < todo; ++t) {
                const int tile = r.tile0 + c.tile + t;
                const int next = t + 1 < todo ? page_of(tile + 1) : -1;
                const int key = tile * kTile + lane * box;
                // keys of the box inside [lo, hi), as bits of the tile's mask
                unsigned long long bits = 0;
                if (page >= 0) {
                    const int from = max(key, r.lo) - tile * kTile, to = min(key + box, r.hi) - tile * kTile;
                    bits = (~0ull >> (64 - (to - from))) << from;
                }
                const uint32_t lo32 = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(bits));
                const uint32_t hi32 = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(bits >> 32));
                const int loads = __popc(__ballot_sync(0xffffffffu, page >= 0));
                ok = ptx::mbar_wait(empty_bar(stage), phase ^ 1u, a.status, 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) {
                    mask_p[stage] = static_cast<unsigned long long>(hi32) << 32 | lo32;
                    ptx::mbar_arrive_expect_tx(full_bar(stage), static_cast<uint32_t>(loads) * box * 2 * (C::kRowBytes + (FP8 ? 4 : 0)));
                }
                __syncwarp();
                if (page >= 0) {
                    const int row = ((page * s.kv_heads + c.h) << s.page_shift) + (key & ((1 << s.page_shift) - 1));
                    const uint32_t to = ring + stage * C::kStageBytes + lane * box * C::kBoxBytes;
#pragma unroll
                    for (int h = 0; h < C::kHalves; ++h) {
                        ptx::tma_load_2d(to + h * C::kHalfBytes, &tmK, full_bar(stage), h * C::kBoxBytes, row);
                        ptx::tma_load_2d(to + C::kTensorBytes + h * C::kHalfBytes, &tmV, full_bar(stage), h * C::kBoxBytes, row);
                    }
                    if (FP8) {
                        const uint32_t sc = ring + stage * C::kStageBytes + 2 * C::kTensorBytes + lane * box * 4;
                        ptx::bulk_load(sc, a.k_scale + row, box * 4, full_bar(stage));
                        ptx::bulk_load(sc + C::kScaleBytes, a.v_scale + row, box * 4, full_bar(stage));
                    }
                }
                __syncwarp();
                page = next;
                if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
            }
            c.at += todo;
            if (c.at < c.end) next_block(s, c, q, kRows);
        }
        if (!ok) __nanosleep(200000);
        return;
    }

    // ---------------------------------------------------------------------------------------------- consumers
    const int g = lane >> 2, cc = lane & 3;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (c.at < c.end) {
        const Range r = block_range(s, q, c.i, kRows, kTile);
        const int todo = static_cast<int>(min(static_cast<long long>(r.tiles - c.tile), c.end - c.at));
        const int r0 = c.i * kRows, rows = min(kRows, q.n * s.group - r0);
        // this thread's two rows: where they stand in q, and their positions
        int pos[2];
        const __nv_bfloat16* qp[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int row = min(g + 8 * u, rows - 1);
            const int t = (r0 + row) / s.group;
            pos[u] = q.kv - q.n + t;
            qp[u] = a.q + (q.q0 + t) * a.q_stride + (c.h * s.group + (r0 + row) - t * s.group) * a.q_head;
        }
        const int pos_lo = __shfl_sync(0xffffffffu, pos[0], 0), pos_hi = __shfl_sync(0xffffffffu, pos[1], 31);
        uint32_t qa[C::kSteps][4];
#pragma unroll
        for (int ks = 0; ks < C::kSteps; ++ks)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint2 w = __ldg(reinterpret_cast<const uint2*>(qp[u] + q_element<D, FP8>(ks, cc)));
                if (FP8) w = make_uint2(__byte_perm(w.x, w.y, 0x5410), __byte_perm(w.x, w.y, 0x7632));     // even and odd elements
                qa[ks][u] = w.x;
                qa[ks][2 + u] = w.y;
            }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float o[C::kCols][4];
#pragma unroll
        for (int i = 0; i < C::kCols; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

        for (int t = 0; t < todo; ++t) {
            if (ok) ok = ptx::mbar_wait(full_bar(stage), phase, a.status, 2);
            const int key0 = (r.tile0 + c.tile + t) * kTile + warp * 16;
            const uint32_t valid = static_cast<uint32_t>(mask_p[stage] >> (16 * warp)) & 0xFFFFu;
            if (ok && valid != 0) {
                const uint32_t kb = ring + stage * C::kStageBytes, vb = kb + C::kTensorBytes;
                float x[2][4] = {};                                  // products with keys 8 * nt + 2 * cc + {0, 1}
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const int row = warp * 16 + nt * 8 + g;
                    if constexpr (FP8) {
#pragma unroll
                        for (int v = 0; v < D / 64; ++v) {
                            const uint4 w = ptx::ld_shared_v4(swizzled<C::kBoxBytes>(kb, row, D == 128 ? (2 * cc + v) * 16 : cc * 16));
                            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t (&qf)[4] = qa[4 * v + i];
                                ptx::mma_bf16_16816(x[nt], qf[0], qf[1], qf[2], qf[3], e4m3x2(ws[i] << 8), e4m3x2(ws[i]));
                            }
                        }
                    } else {
#pragma unroll
                        for (int hv = 0; hv < D / 32; ++hv) {
                            const uint4 w = ptx::ld_shared_v4(swizzled<128>(kb + (hv >> 1) * C::kHalfBytes, row, (2 * cc + (hv & 1)) * 16));
                            const uint32_t (&q0)[4] = qa[2 * hv];
                            const uint32_t (&q1)[4] = qa[2 * hv + 1];
                            ptx::mma_bf16_16816(x[nt], q0[0], q0[1], q0[2], q0[3], w.x, w.y);
                            ptx::mma_bf16_16816(x[nt], q1[0], q1[1], q1[2], q1[3], w.z, w.w);
                        }
                    }
                }
                // scores in units of log2; a key's scale first
                float vs[2][2];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    float2 ks = make_float2(1.0f, 1.0f), v2 = ks;
                    if (FP8) {
                        const uint32_t at = kb + 2 * C::kTensorBytes + (warp * 16 + nt * 8 + 2 * cc) * 4;
                        const uint2 w = ptx::ld_shared_v2(at), y = ptx::ld_shared_v2(at + C::kScaleBytes);
                        ks = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
                        v2 = make_float2(__uint_as_float(y.x), __uint_as_float(y.y));
                    }
                    vs[nt][0] = v2.x; vs[nt][1] = v2.y;
                    const float f0 = ks.x * a.scale_log2, f1 = ks.y * a.scale_log2;
                    x[nt][0] *= f0; x[nt][1] *= f1; x[nt][2] *= f0; x[nt][3] *= f1;
                }
                // keys that are not there for the whole block (their values are zeroed too: what lies in their place may
                // be anything), that come after a row, or that have left its window
                const bool whole = valid == 0xFFFFu && (!s.causal || key0 + 15 <= pos_lo) && (s.window == 0 || key0 > pos_hi - s.window);
                if (!whole) {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int j = nt * 8 + 2 * cc + e;
                            const bool there = (valid >> j) & 1u;
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const int key = key0 + j;
                                const bool seen = there && (!s.causal || key <= pos[u]) && (s.window == 0 || key > pos[u] - s.window);
                                if (!seen) x[nt][2 * u + e] = -INFINITY;
                            }
                        }
                }
                uint32_t pa[4];
                float f[2];
                bool moved = false;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float t4 = max_nan4(x[0][2 * u], x[0][2 * u + 1], x[1][2 * u], x[1][2 * u + 1]);
                    t4 = ptx::max_nan(t4, __shfl_xor_sync(0xffffffffu, t4, 1));
                    t4 = ptx::max_nan(t4, __shfl_xor_sync(0xffffffffu, t4, 2));
                    const float mn = ptx::max_nan(m[u], t4);
                    const float base = mn == -INFINITY ? 0.0f : mn;          // a row that has seen nothing yet
                    f[u] = ptx::ex2(m[u] - base);
                    moved |= mn != m[u];
                    m[u] = mn;
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] = ptx::ex2(x[i >> 1][2 * u + (i & 1)] - base);
                    l[u] = l[u] * f[u] + ((p[0] + p[1]) + (p[2] + p[3]));
                    if (FP8) {
                        // a masked key's p is 0: its product with a scale that is not finite must be 0 as well
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[i] = !whole && p[i] == 0.0f ? 0.0f : p[i] * vs[i >> 1][i & 1];
                    }
                    pa[u] = pack_bf16x2(p[0], p[1]);
                    pa[2 + u] = pack_bf16x2(p[2], p[3]);
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int i = 0; i < C::kCols; ++i) { o[i][0] *= f[0]; o[i][1] *= f[0]; o[i][2] *= f[1]; o[i][3] *= f[1]; }
                }
                // values: thread (g, cc) takes columns of chunk g in rows 2cc, 2cc+1, 2cc+8, 2cc+9
                const int vr = warp * 16 + 2 * cc;
                const uint32_t keep[4] = {(valid >> (2 * cc)) & 1u, (valid >> (2 * cc + 1)) & 1u, (valid >> (2 * cc + 8)) & 1u, (valid >> (2 * cc + 9)) & 1u};
                if constexpr (FP8) {
                    uint32_t w[4][D / 32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = vr + (i & 1) + 8 * (i >> 1);
                        if constexpr (D == 128) {
                            const uint4 y = ptx::ld_shared_v4(swizzled<128>(vb, row, g * 16));
                            w[i][0] = y.x; w[i][1] = y.y; w[i][2] = y.z; w[i][3] = y.w;
                        } else {
                            const uint2 y = ptx::ld_shared_v2(swizzled<64>(vb, row, g * 8));
                            w[i][0] = y.x; w[i][1] = y.y;
                        }
                    }                                                 // bytes are finite whatever they are: no need to zero them
#pragma unroll
                    for (int j = 0; j < D / 32; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t sel = (e << 4) | ((4 + e) << 12);
                            ptx::mma_bf16_16816(o[4 * j + e], pa[0], pa[1], pa[2], pa[3], e4m3x2(__byte_perm(w[0][j], w[1][j], sel)),
                                                e4m3x2(__byte_perm(w[2][j], w[3][j], sel)));
                        }
                } else {
#pragma unroll
                    for (int h = 0; h < C::kHalves; ++h) {
                        uint32_t w[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 y = ptx::ld_shared_v4(swizzled<128>(vb + h * C::kHalfBytes, vr + (i & 1) + 8 * (i >> 1), g * 16));
                            const bool in = whole || keep[i];
                            w[i][0] = in ? y.x : 0u; w[i][1] = in ? y.y : 0u; w[i][2] = in ? y.z : 0u; w[i][3] = in ? y.w : 0u;
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            ptx::mma_bf16_16816(o[8 * h + 2 * j], pa[0], pa[1], pa[2], pa[3], __byte_perm(w[0][j], w[1][j], 0x5410),
                                                __byte_perm(w[2][j], w[3][j], 0x5410));
                            ptx::mma_bf16_16816(o[8 * h + 2 * j + 1], pa[0], pa[1], pa[2], pa[3], __byte_perm(w[0][j], w[1][j], 0x7632),
                                                __byte_perm(w[2][j], w[3][j], 0x7632));
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(empty_bar(stage));
            if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }

        // ------------------------------------------------------------------------ the four warps' states become one
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
            if (cc == 0) state_p[warp * kRows + g + 8 * u] = make_float2(m[u], l[u]);
        }
        ptx::named_barrier(1, 32 * kConsumers);
        float mm[2], ll[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float2 st[kConsumers];
            mm[u] = -INFINITY;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) { st[w] = state_p[w * kRows + g + 8 * u]; mm[u] = ptx::max_nan(mm[u], st[w].x); }
            const float base = mm[u] == -INFINITY ? 0.0f : mm[u];
            ll[u] = 0.0f;
#pragma unroll
            for (int w = 0; w < kConsumers; ++w) ll[u] += st[w].y * ptx::ex2(st[w].x - base);
            const float f = ptx::ex2(m[u] - base);
#pragma unroll
            for (int i = 0; i < C::kCols; ++i) { o[i][2 * u] *= f; o[i][2 * u + 1] *= f; }
        }
#pragma unroll
        for (int w = kConsumers - 1; w >= 1; --w) {                  // one after the other they hand over to warp 0
            if (warp == w) {
#pragma unroll
                for (int i = 0; i < C::kCols; ++i)
                    *reinterpret_cast<float4*>(join_p + i * 128 + lane * 4) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
            }
            ptx::named_barrier(1, 32 * kConsumers);
            if (warp == 0) {
#pragma unroll
                for (int i = 0; i < C::kCols; ++i) {
                    const float4 y = *reinterpret_cast<const float4*>(join_p + i * 128 + lane * 4);
                    o[i][0] += y.x; o[i][1] += y.y; o[i][2] += y.z; o[i][3] += y.w;
                }
            }
            if (w > 1) ptx::named_barrier(1, 32 * kConsumers);       // before the buffer is written again
        }
        if (warp == 0) {
            const bool begins = c.tile == 0, ends = c.tile + todo == r.tiles;
            // column of accumulator i, element e: thread cc holds columns 2cc + e of group i
            auto column = [&](int i, int e) {
                if (FP8) return (2 * cc + e) * (D / 8) + i;
                return (i >> 3) * 64 + (2 * cc + e) * 8 + (i & 7);
            };
            if (begins && ends) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int row = g + 8 * u;
                    if (row >= rows) continue;
                    const int t = (r0 + row) / s.group;
                    const size_t to = static_cast<size_t>(q.q0 + t) * s.heads + c.h * s.group + (r0 + row) - t * s.group;
                    const float inv = ll[u] == 0.0f ? 0.0f : __frcp_rn(ll[u]);
                    // column(i, e) is contiguous in i over runs of 8 (or 16)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < C::kCols; i += 8) {
                            uint4 w;
                            w.x = pack_bf16x2(o[i][2 * u + e] * inv, o[i + 1][2 * u + e] * inv);
                            w.y = pack_bf16x2(o[i + 2][2 * u + e] * inv, o[i + 3][2 * u + e] * inv);
                            w.z = pack_bf16x2(o[i + 4][2 * u + e] * inv, o[i + 5][2 * u + e] * inv);
                            w.w = pack_bf16x2(o[i + 6][2 * u + e] * inv, o[i + 7][2 * u + e] * inv);
                            *reinterpret_cast<uint4*>(a.out + to * D + column(i, e)) = w;
                        }
                    if (a.lse != nullptr && cc == 0) a.lse[to] = lse_of(mm[u], ll[u]);
                }
            } else {
                const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
                float* po = a.part + static_cast<size_t>(slot) * kRows * (D + 2);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int row = g + 8 * u;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < C::kCols; i += 4)
                            *reinterpret_cast<float4*>(po + row * D + column(i, e)) =
                                make_float4(o[i][2 * u + e], o[i + 1][2 * u + e], o[i + 2][2 * u + e], o[i + 3][2 * u + e]);
                    if (cc == 0) *reinterpret_cast<float2*>(po + kRows * D + row * 2) = make_float2(mm[u], ll[u]);
                }
                if (begins && lane == 0) {
                    Open* op = a.open + blockIdx.x;
                    op->token0 = q.q0; op->r0 = r0; op->rows = rows; op->h = c.h;
                    op->last = owner(c, c.at + r.tiles - 1);
                }
            }
        }
        ptx::named_barrier(1, 32 * kConsumers);                       // the state and the join buffer are free again
        c.at += todo;
        if (c.at < c.end) next_block(s, c, q, kRows);
    }
}

template <int D, bool FP8>
int launch(const Args& args, cudaStream_t stream)
{
    using C = Cfg<D, FP8>;
    Args a = args;
    const int box = kTile < (1 << a.s.page_shift) ? kTile : 1 << a.s.page_shift;
    const uint64_t rows = (static_cast<uint64_t>(a.s.num_pages) * a.s.kv_heads) << a.s.page_shift;
    CUtensorMap tmK, tmV;
    const CUtensorMapSwizzle sw = C::kBoxBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    if (!make_tmap_2d_u8(&tmK, a.k_cache, rows, C::kRowBytes, C::kRowBytes, box, C::kBoxBytes, sw)) return cudaErrorInvalidValue;
    if (!make_tmap_2d_u8(&tmV, a.v_cache, rows, C::kRowBytes, C::kRowBytes, box, C::kBoxBytes, sw)) return cudaErrorInvalidValue;
    auto kernel = attn_split_kernel<D, FP8>;
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured[dev] = true;
    }
    if (static_cast<long long>(a.s.seqs) * 8 > C::kStages * C::kStageBytes) return cudaErrorInvalidValue;
    a.block_limit = static_cast<int>((static_cast<long long>(a.max_q) * a.s.group + kRows - 1) / kRows);
    const int ctas = 2 * num_sms();
    kernel<<<ctas, kThreads, C::kSmemBytes, stream>>>(tmK, tmV, a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_combine<D>(a, ctas, kRows, stream);
}

}  // namespace split

int attn_split(const Args& a, int head_dim, bool fp8, cudaStream_t stream)
{
    if (head_dim == 64) return fp8 ? split::launch<64, true>(a, stream) : split::launch<64, false>(a, stream);
    return fp8 ? split::launch<128, true>(a, stream) : split::launch<128, false>(a, stream);
}

size_t attn_split_workspace(int head_dim)
{
    return static_cast<size_t>(2 * num_sms()) * (2 * split::kRows * (head_dim + 2) * sizeof(float) + sizeof(Open)) + 32;
}

}  // namespace paged
}  // namespace b200q
