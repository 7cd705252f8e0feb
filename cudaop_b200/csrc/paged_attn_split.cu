// Attention of a chunk of new tokens over a paged cache, for few rows per kv head (decode, drafted tokens): the split-KV
// kernel.
//
//   o[r,:] = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x_j = scale * log2(e) * (q_r . k_j),  m = max_j x_j
// over the keys j that row r sees.
//
// Bound by the bytes of the cache: one pass over the keys, meant to run at HBM rate.  A CTA is a producer warp that fills a ring of
// 64-key tiles by TMA (one box per page and tensor; the page table is read a tile ahead) and four consumer warps of 16
// keys each: their softmax states are independent, so a tile needs no barrier but the ring's, and they meet once per block of rows.
// The products are computed transposed, keys (then head_dim) on the 16 side of m16n8k16 and 8 rows on its narrow side: with 8
// query heads per kv head a decode step fills it exactly (rows on the 16 side left half of the products, of the softmax
// and of the accumulator registers to rows that do not exist: 571 instructions per 16 keys of 128 against 367, and
// 247 us against 149 us for 48 sequences of 1 to 16 thousand tokens, 8 kv heads, E4M3).  Between the two products the 8x8 blocks of p are
// transposed in registers (movmatrix).  The order of the contraction over head_dim, and of the output columns, is permuted so that
// every shared-memory read is a conflict-free 16 (or 8) byte load of consecutive elements.
//
// Precision.  An E4M3 cache is never rounded again: the bytes become fp16 exactly, a key's scale multiplies the 32-bit
// product q.k, and a value's scale multiplies p.  The fp16 operands are kept in range by powers of two: a row of q is divided
// by that of its largest element (an element 2^15 below it starts to lose bits that are below those of the 32-bit sum), and p * scale by that of
// its own running maximum over the keys that the row sees (paged_common.cuh).  So it keeps 11 bits.  A bf16 cache needs bf16 operands, which would leave p 8
// bits; it is split in two (its rounding and the rest) and the second product runs twice, which costs nothing here.
// Sums, maxima and accumulators are 32-bit.  The work is divided over the persistent grid by tiles (paged_common.cuh).
#include "paged_common.cuh"
#include "paged_attn.cuh"
#include "ptx.cuh"
#include <cfloat>

namespace b200q {
namespace paged {
namespace split {

constexpr int kTile = 64, kConsumers = 4, kThreads = 32 * (kConsumers + 1);

// NT: groups of 8 rows per block
template <int D, bool FP8, int NT>
struct Cfg {
    static constexpr int kRows = 8 * NT;
    static constexpr int kCtasPerSm = NT == 1 ? 3 : 2;
    static constexpr int kRowBytes = FP8 ? D : 2 * D;
    static constexpr int kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;       // inner extent of a box = swizzle span
    static constexpr int kHalves = kRowBytes / kBoxBytes;
    static constexpr int kHalfBytes = kTile * kBoxBytes;
    static constexpr int kTensorBytes = kTile * kRowBytes;
    static constexpr int kScaleBytes = FP8 ? kTile * 4 : 0;
    static constexpr int kStageBytes = (2 * kTensorBytes + 2 * kScaleBytes + 1023) / 1024 * 1024;
    static constexpr int kJoinBytes = kRows * D * 4;                          // one warp's accumulators
    static constexpr int kBudget = 227 * 1024 / kCtasPerSm - 1024 - 1024 - 768 - kJoinBytes;     // (1 KB the system keeps, 1 KB to align, states)
    static constexpr int kStages = kBudget / kStageBytes < 8 ? kBudget / kStageBytes : 8;
    static_assert(kStages >= 2, "ring");
    static_assert(kStages * kStageBytes >= 8192 * 4, "a word per sequence");
    static constexpr int kStateBytes = kConsumers * kRows * 8;                // running maximum and sum per warp and row
    static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kJoinBytes + kStateBytes + kStages * (8 + 16);
    static constexpr int kSteps = D / 16;                                     // k-steps of q.k, and 16-column groups of the output
};

// The row of q as 16-bit elements in the order the products take them: k-step s gives thread c = lane % 4 the four
// consecutive elements that follow q_element(s, c).
template <int D, bool FP8>
__device__ __forceinline__ int q_element(int s, int c)
{
    if (FP8) return D == 128 ? (2 * c + (s >> 2)) * 16 + 4 * (s & 3) : c * 16 + 4 * s;
    return (s >> 2) * 64 + (2 * c + ((s >> 1) & 1)) * 8 + 4 * (s & 1);
}

// byte `byte` of row `row` of a tile half whose rows are kBox bytes, 128- (64-) byte swizzle
template <int kBox>
__device__ __forceinline__ uint32_t swizzled(uint32_t base, int row, int byte)
{
    const uint32_t a = static_cast<uint32_t>(row) * kBox + byte;
    return base + (a ^ (kBox == 128 ? (a >> 3) & 0x70u : (a >> 3) & 0x30u));
}

// Adds the values of a half tile's 16 keys that are not finite to the rows that see them; `at`: the first of the warp's rows, whose
// eight 16-byte units are swizzled; a lane has columns of unit g.  Rare, and short rather than fast.
template <int NT, int STEPS, typename Seen>
__device__ __forceinline__ void add_not_finite(float (&o)[NT][STEPS][4], int h, uint32_t at, int g, uint32_t valid, Seen seen)
{
#pragma unroll 1
    for (int j = 0; j < 16; ++j) {
        if (!((valid >> j) & 1u)) continue;
        const uint4 y = ptx::ld_shared_v4(at + j * 128 + ((g ^ (j & 7)) << 4));
        const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = __uint_as_float(e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
            const bool odd = (__float_as_uint(v) & 0x7F800000u) == 0x7F800000u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int hh = 0; hh < STEPS / 4; ++hh)
                        if (hh == h && odd && seen(j, nt, u)) o[nt][4 * hh + (e >> 1)][2 * (e & 1) + u] += v;
        }
    }
}

template <bool FP8>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if (FP8) ptx::mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
    else ptx::mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
}

template <int D, bool FP8, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2)
attn_split_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Args a)
{
    using C = Cfg<D, FP8, NT>;
    constexpr int kRows = C::kRows;
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
    Cursor c = find_work(s, kRows, kTile, reinterpret_cast<int*>(smem_raw + (ring - raw)), a.block_limit, a.block_most, blockIdx.x, gridDim.x);
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
            const int todo = min(r.tiles - c.tile, c.end - c.at);
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
    // lane 4g + cc: keys g and g + 8 of the warp's 16, rows 8 * nt + 2cc + {0, 1} (and, of the output, columns of chunk g)
    const int g = lane >> 2, cc = lane & 3;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (c.at < c.end) {
        const Range r = block_range(s, q, c.i, kRows, kTile);
        const int todo = min(r.tiles - c.tile, c.end - c.at);
        const int r0 = c.i * kRows, rows = min(kRows, q.n * s.group - r0);
        // q: this thread holds row 8 * nt + g; what belongs to rows 2cc + {0, 1} comes from the lanes that hold them
        uint32_t qb[NT][C::kSteps][2];
        int pos[NT][2];
        float row_scale[NT][2];                                      // softmax scale (and, for fp16 rows, their power of two)
        int pos_lo = 0, pos_hi = 0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = min(8 * nt + g, rows - 1);               // rows behind the block repeat its last one
            const int t = s.token_of(r0 + row);
            const __nv_bfloat16* qp = a.q + (q.q0 + t) * a.q_stride + (c.h * s.group + (r0 + row) - t * s.group) * a.q_head;
#pragma unroll
            for (int ks = 0; ks < C::kSteps; ++ks) {
                const uint2 w = __ldg(reinterpret_cast<const uint2*>(qp + q_element<D, FP8>(ks, cc)));
                qb[nt][ks][0] = w.x;
                qb[nt][ks][1] = w.y;
            }
            float factor = a.scale_log2;
            if (FP8) {
                uint32_t m2 = 0;
#pragma unroll
                for (int ks = 0; ks < C::kSteps; ++ks) m2 = __vmaxu2(m2, __vmaxu2(qb[nt][ks][0] & 0x7FFF7FFFu, qb[nt][ks][1] & 0x7FFF7FFFu));
                uint32_t mx = max(m2 & 0xFFFFu, m2 >> 16);
                mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const uint32_t e = min(max(mx >> 7, 1u), 253u);      // exponent field of the largest element
                const float down = pow2_of_field(254u - e);          // 2^(127 - e): the row's largest element becomes 1 to 4
                factor *= pow2_of_field(e);
#pragma unroll
                for (int ks = 0; ks < C::kSteps; ++ks)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t w = qb[nt][ks][i];
                        qb[nt][ks][i] = pack_f16x2(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xFFFF0000u) * down);
                    }
            }
            const int p = q.kv - q.n + t;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                pos[nt][u] = __shfl_sync(0xffffffffu, p, 4 * (2 * cc + u));
                row_scale[nt][u] = __shfl_sync(0xffffffffu, factor, 4 * (2 * cc + u));
            }
            if (nt == 0) pos_lo = __shfl_sync(0xffffffffu, p, 0);
            pos_hi = __shfl_sync(0xffffffffu, p, 31);
        }
        float m[NT][2], l[NT][2], n[NT][2], o[NT][C::kSteps][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int u = 0; u < 2; ++u) { m[nt][u] = -INFINITY; n[nt][u] = -FLT_MAX; l[nt][u] = 0.0f; }
#pragma unroll
            for (int i = 0; i < C::kSteps; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
        }

        for (int t = 0; t < todo; ++t) {
            if (ok) ok = ptx::mbar_wait(full_bar(stage), phase, a.status, 2);
            const int key0 = (r.tile0 + c.tile + t) * kTile + warp * 16;
            const uint32_t valid = static_cast<uint32_t>(mask_p[stage] >> (16 * warp)) & 0xFFFFu;
            if (ok && valid != 0) {
                const uint32_t kb = ring + stage * C::kStageBytes, vb = kb + C::kTensorBytes;
                const int kr = warp * 16 + g;
                float x[NT][4];                                      // keys g (0, 1) and g + 8 (2, 3) with rows 2cc + {0, 1}
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.0f;
                if constexpr (FP8) {
#pragma unroll
                    for (int v = 0; v < D / 64; ++v) {
                        const int byte = D == 128 ? (2 * cc + v) * 16 : cc * 16;
                        const uint4 w = ptx::ld_shared_v4(swizzled<C::kBoxBytes>(kb, kr, byte)), y = ptx::ld_shared_v4(swizzled<C::kBoxBytes>(kb, kr + 8, byte));
                        const uint32_t ws[4] = {w.x, w.y, w.z, w.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t a0 = ptx::e4m3x2_lo(ws[i]), a1 = ptx::e4m3x2_lo(ys[i]), a2 = ptx::e4m3x2_hi(ws[i]), a3 = ptx::e4m3x2_hi(ys[i]);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma<FP8>(x[nt], a0, a1, a2, a3, qb[nt][4 * v + i][0], qb[nt][4 * v + i][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int hv = 0; hv < D / 32; ++hv) {
                        const uint32_t half = kb + (hv >> 1) * C::kHalfBytes;
                        const int byte = (2 * cc + (hv & 1)) * 16;
                        const uint4 w = ptx::ld_shared_v4(swizzled<128>(half, kr, byte)), y = ptx::ld_shared_v4(swizzled<128>(half, kr + 8, byte));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma<FP8>(x[nt], w.x, y.x, w.y, y.y, qb[nt][2 * hv][0], qb[nt][2 * hv][1]);
                            mma<FP8>(x[nt], w.z, y.z, w.w, y.w, qb[nt][2 * hv + 1][0], qb[nt][2 * hv + 1][1]);
                        }
                    }
                }
                float ks[2] = {1.0f, 1.0f}, vs[2] = {1.0f, 1.0f};    // of keys g and g + 8
                const bool there[2] = {((valid >> g) & 1u) != 0, ((valid >> (g + 8)) & 1u) != 0};
                float ve[2] = {0.0f, 0.0f};                          // log2 of the powers of two above the value scales
                if (FP8) {
                    const uint32_t at = kb + 2 * C::kTensorBytes + kr * 4;
                    ks[0] = ptx::ld_shared_f32(at); ks[1] = ptx::ld_shared_f32(at + 32);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float v = ptx::ld_shared_f32(at + C::kScaleBytes + 32 * k);
                        ve[k] = log2_above(field_of(v));
                        vs[k] = mantissa_of(v);
                    }
                }
                // keys that are not there for the whole block, that come after a row, or that have left its window
                const bool whole = valid == 0xFFFFu && (!s.causal || key0 + 15 <= pos_lo) && (s.window == 0 || key0 > pos_hi - s.window);
                uint32_t pb[NT][2], pl[NT][2];
                bool moved = false;
                float f[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = i >> 1, u = i & 1;
                        x[nt][i] *= FP8 ? ks[k] * row_scale[nt][u] : row_scale[nt][u];
                        if (!whole) {
                            const int key = key0 + g + 8 * k;
                            const bool seen = there[k] && (!s.causal || key <= pos[nt][u]) && (s.window == 0 || key > pos[nt][u] - s.window);
                            if (!seen) x[nt][i] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float mn = ptx::max_nan(x[nt][u], x[nt][2 + u]);
#pragma unroll
                        for (int w = 4; w <= 16; w <<= 1) mn = ptx::max_nan(mn, __shfl_xor_sync(0xffffffffu, mn, w));
                        mn = ptx::max_nan(mn, m[nt][u]);
                        const float base = mn == -INFINITY ? 0.0f : mn;      // a row that has seen nothing yet
                        const float fm = ptx::ex2(m[nt][u] - base);
                        f[nt][u] = fm;
                        moved |= !FP8 && mn != m[nt][u];
                        p[u] = ptx::ex2(x[nt][u] - base);
                        p[2 + u] = ptx::ex2(x[nt][2 + u] - base);
                        l[nt][u] = l[nt][u] * fm + (p[u] + p[2 + u]);
                        m[nt][u] = mn;
                        if (FP8) {                                   // from here on x + e
                            x[nt][u] += ve[0];
                            x[nt][2 + u] += ve[1];
                            moved |= fmaxf(x[nt][u], x[nt][2 + u]) > n[nt][u] + kLazy;
                        }
                    }
                    if (!FP8) {
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t hi = pack_bf16x2(p[2 * k], p[2 * k + 1]);
                            pl[nt][k] = ptx::movmatrix_trans(pack_bf16x2(p[2 * k] - __uint_as_float(hi << 16), p[2 * k + 1] - __uint_as_float(hi & 0xFFFF0000u)));
                            pb[nt][k] = ptx::movmatrix_trans(hi);
                        }
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
                    if (FP8) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                float nn = fmaxf(x[nt][u], x[nt][2 + u]);
#pragma unroll
                                for (int w = 4; w <= 16; w <<= 1) nn = fmaxf(nn, __shfl_xor_sync(0xffffffffu, nn, w));
                                nn = fmaxf(nn, n[nt][u]);
                                f[nt][u] = nn == n[nt][u] ? 1.0f : ptx::ex2(n[nt][u] - nn);
                                n[nt][u] = nn;
                            }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < C::kSteps; ++i) { o[nt][i][0] *= f[nt][0]; o[nt][i][1] *= f[nt][1]; o[nt][i][2] *= f[nt][0]; o[nt][i][3] *= f[nt][1]; }
                }
                if (FP8) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float p[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[i] = ptx::ex2(x[nt][i] + (kRoomLog2 - n[nt][i & 1])) * vs[i >> 1];
                            // a key that the row does not see: its scale may be anything
                            if (!whole && x[nt][i] == -INFINITY) p[i] = 0.0f;
                        }
                        pb[nt][0] = ptx::movmatrix_trans(pack_f16x2(p[0], p[1]));
                        pb[nt][1] = ptx::movmatrix_trans(pack_f16x2(p[2], p[3]));
                    }
                }
                // values: columns of chunk g in rows 2cc, 2cc + 1, 2cc + 8, 2cc + 9; what is not there counts as zero, whatever it is
                const int vr = warp * 16 + 2 * cc;
                bool in[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) in[i] = whole || ((valid >> (2 * cc + (i & 1) + 8 * (i >> 1))) & 1u);
                if constexpr (FP8) {
                    uint32_t w[4][D / 32];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = vr + (i & 1) + 8 * (i >> 1);
                        if constexpr (D == 128) {
                            const uint4 y = ptx::ld_shared_v4(swizzled<128>(vb, row, g * 16));
                            w[i][0] = in[i] ? y.x : 0u; w[i][1] = in[i] ? y.y : 0u; w[i][2] = in[i] ? y.z : 0u; w[i][3] = in[i] ? y.w : 0u;
                        } else {
                            const uint2 y = ptx::ld_shared_v2(swizzled<64>(vb, row, g * 8));
                            w[i][0] = in[i] ? y.x : 0u; w[i][1] = in[i] ? y.y : 0u;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < D / 32; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {                // columns 4j + 2e, 4j + 2e + 1 of the chunk
                            const uint32_t sel = e == 0 ? 0x5140u : 0x7362u;
                            const uint32_t lo = __byte_perm(w[0][j], w[1][j], sel), hi = __byte_perm(w[2][j], w[3][j], sel);
                            const uint32_t a0 = ptx::e4m3x2_lo(lo), a1 = ptx::e4m3x2_hi(lo), a2 = ptx::e4m3x2_lo(hi), a3 = ptx::e4m3x2_hi(hi);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma<FP8>(o[nt][2 * j + e], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                        }
                } else {
#pragma unroll
                    for (int h = 0; h < C::kHalves; ++h) {
                        uint32_t w[4][4], top = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4 y = ptx::ld_shared_v4(swizzled<128>(vb + h * C::kHalfBytes, vr + (i & 1) + 8 * (i >> 1), g * 16));
                            w[i][0] = in[i] ? y.x : 0u; w[i][1] = in[i] ? y.y : 0u; w[i][2] = in[i] ? y.z : 0u; w[i][3] = in[i] ? y.w : 0u;
#pragma unroll
                            for (int j = 0; j < 4; ++j) top = __vmaxu2(top, w[i][j] & 0x7FFF7FFFu);
                        }
                        if (__any_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16) >= 0x7F80u)) {
                            // Values that are not finite: a product would carry them, as 0 * infinity, into the rows that do not see
                            // their key (and turn an infinity into NaN by the second term of p).  They are added by themselves.
                            add_not_finite<NT>(o, h, swizzled<128>(vb + h * C::kHalfBytes, warp * 16, 0), g, valid,
                                               [&](int j, int nt, int u) {
                                                   const int key = key0 + j;
                                                   return (!s.causal || key <= pos[nt][u]) && (s.window == 0 || key > pos[nt][u] - s.window);
                                               });
#pragma unroll
                            for (int i = 0; i < 4; ++i)
#pragma unroll
                                for (int j = 0; j < 4; ++j) w[i][j] = only_finite(w[i][j]);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t a0 = __byte_perm(w[0][j], w[1][j], 0x5410), a1 = __byte_perm(w[0][j], w[1][j], 0x7632);
                            const uint32_t a2 = __byte_perm(w[2][j], w[3][j], 0x5410), a3 = __byte_perm(w[2][j], w[3][j], 0x7632);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma<FP8>(o[nt][4 * h + j], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                                mma<FP8>(o[nt][4 * h + j], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
                            }
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
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int w = 4; w <= 16; w <<= 1) l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], w);
                if (g == 0) state_p[warp * kRows + 8 * nt + 2 * cc + u] = make_float2(m[nt][u], l[nt][u]);
            }
        ptx::named_barrier(1, 32 * kConsumers);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float2 st[kConsumers];
                float mm = -INFINITY, ll = 0.0f;
#pragma unroll
                for (int w = 0; w < kConsumers; ++w) { st[w] = state_p[w * kRows + 8 * nt + 2 * cc + u]; mm = ptx::max_nan(mm, st[w].x); }
                const float base = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
                for (int w = 0; w < kConsumers; ++w) ll += st[w].y * ptx::ex2(st[w].x - base);
                // E4M3: from the units of n, in two steps, since 2^(n - base) alone may lie outside the range of the numbers
                const float fw = FP8 ? ptx::ex2(0.5f * (n[nt][u] - base)) : ptx::ex2(m[nt][u] - base), fw2 = fw * kRoomInv;
#pragma unroll
                for (int i = 0; i < C::kSteps; ++i) {
                    o[nt][i][u] *= fw; o[nt][i][2 + u] *= fw;
                    if (FP8) { o[nt][i][u] *= fw2; o[nt][i][2 + u] *= fw2; }
                }
                m[nt][u] = mm;
                l[nt][u] = ll;
            }
#pragma unroll
        for (int w = kConsumers - 1; w >= 1; --w) {                  // one after the other they hand over to warp 0
            if (warp == w) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < C::kSteps; ++i)
                        *reinterpret_cast<float4*>(join_p + (nt * C::kSteps + i) * 128 + lane * 4) = make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]);
            }
            ptx::named_barrier(1, 32 * kConsumers);
            if (warp == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < C::kSteps; ++i) {
                        const float4 y = *reinterpret_cast<const float4*>(join_p + (nt * C::kSteps + i) * 128 + lane * 4);
                        o[nt][i][0] += y.x; o[nt][i][1] += y.y; o[nt][i][2] += y.z; o[nt][i][3] += y.w;
                    }
            }
            if (w > 1) ptx::named_barrier(1, 32 * kConsumers);       // before the buffer is written again
        }
        if (warp == 0) {
            const bool begins = c.tile == 0, ends = c.tile + todo == r.tiles;
            // accumulator group i, element 2 * e + u: row 2cc + u, column 2i + e of chunk g (16 columns of an E4M3 row of 128,
            // else 8; group 4h + j of a bf16 row is columns 2j, 2j + 1 of half h)
            constexpr int kRun = FP8 && D == 128 ? 16 : 8;
            const int slot = 2 * blockIdx.x + (begins ? 1 : 0);
            float* po = a.part + static_cast<size_t>(slot) * kRows * (D + 2);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int row = 8 * nt + 2 * cc + u;
                    if (begins && ends) {
                        if (row >= rows) continue;
                        const int t = s.token_of(r0 + row);
                        const size_t to = static_cast<size_t>(q.q0 + t) * s.heads + c.h * s.group + (r0 + row) - t * s.group;
                        const float inv = l[nt][u] == 0.0f ? 0.0f : __frcp_rn(l[nt][u]);
#pragma unroll
                        for (int i = 0; i < C::kSteps; i += 4) {     // eight columns
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) w[k] = pack_bf16x2(o[nt][i + k][u] * inv, o[nt][i + k][2 + u] * inv);
                            const int col = kRun == 16 ? g * 16 + 2 * i : (i >> 2) * 64 + g * 8;
                            *reinterpret_cast<uint4*>(a.out + to * D + col) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        if (a.lse != nullptr && g == 0) a.lse[to] = lse_of(m[nt][u], l[nt][u]);
                    } else {
#pragma unroll
                        for (int i = 0; i < C::kSteps; i += 2) {
                            const int col = kRun == 16 ? g * 16 + 2 * i : (i >> 2) * 64 + g * 8 + 2 * (i & 3);
                            *reinterpret_cast<float4*>(po + row * D + col) = make_float4(o[nt][i][u], o[nt][i][2 + u], o[nt][i + 1][u], o[nt][i + 1][2 + u]);
                        }
                        if (g == 0) *reinterpret_cast<float2*>(po + kRows * D + row * 2) = make_float2(m[nt][u], l[nt][u]);
                    }
                }
            if (begins && !ends && lane == 0) {
                Open* op = a.open + blockIdx.x;
                op->token0 = q.q0; op->r0 = r0; op->rows = rows; op->h = c.h;
                op->last = owner(c, c.at + r.tiles - 1);
            }
        }
        ptx::named_barrier(1, 32 * kConsumers);                       // the state and the join buffer are free again
        c.at += todo;
        if (c.at < c.end) next_block(s, c, q, kRows);
    }
}

template <int D, bool FP8, int NT>
int launch(const Args& args, cudaStream_t stream)
{
    using C = Cfg<D, FP8, NT>;
    Args a = args;
    const int box = kTile < (1 << a.s.page_shift) ? kTile : 1 << a.s.page_shift;
    const uint64_t rows = (static_cast<uint64_t>(a.s.num_pages) * a.s.kv_heads) << a.s.page_shift;
    CUtensorMap tmK, tmV;
    const CUtensorMapSwizzle sw = C::kBoxBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    if (!make_tmap_2d_u8(&tmK, a.k_cache, rows, C::kRowBytes, C::kRowBytes, box, C::kBoxBytes, sw)) return cudaErrorInvalidValue;
    if (!make_tmap_2d_u8(&tmV, a.v_cache, rows, C::kRowBytes, C::kRowBytes, box, C::kBoxBytes, sw)) return cudaErrorInvalidValue;
    auto kernel = attn_split_kernel<D, FP8, NT>;
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured[dev] = true;
    }
    if (!tiles_fit(a, C::kRows, kTile)) return cudaErrorInvalidValue;
    a.block_limit = static_cast<int>((static_cast<long long>(a.max_q) * a.s.group + C::kRows - 1) / C::kRows);
    a.block_most = static_cast<int>(most_blocks(a, C::kRows));          // (tiles_fit bounds it)
    const int ctas = C::kCtasPerSm * num_sms();
    kernel<<<ctas, kThreads, C::kSmemBytes, stream>>>(tmK, tmV, a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_combine<D>(a, ctas, C::kRows, stream);
}

template <int D, bool FP8>
int launch_rows(const Args& a, cudaStream_t stream)
{
    return static_cast<long long>(a.max_q) * a.s.group <= 8 ? launch<D, FP8, 1>(a, stream) : launch<D, FP8, 2>(a, stream);
}

}  // namespace split

int attn_split(const Args& a, int head_dim, bool fp8, cudaStream_t stream)
{
    if (head_dim == 64) return fp8 ? split::launch_rows<64, true>(a, stream) : split::launch_rows<64, false>(a, stream);
    return fp8 ? split::launch_rows<128, true>(a, stream) : split::launch_rows<128, false>(a, stream);
}

// the larger of 3 CTAs an SM with 8 rows and 2 with 16
int attn_split_ctas() { return 3 * num_sms(); }
size_t attn_split_part_bytes(int head_dim) { return static_cast<size_t>(2 * num_sms()) * 2 * 16 * (head_dim + 2) * sizeof(float); }

}  // namespace paged
}  // namespace b200q
