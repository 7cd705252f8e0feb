// Attention of a chunk of new tokens over a paged cache, for many rows per kv head (prefill in chunks): the tensor-core kernel.
// The mathematics, the division of the work and the treatment of an E4M3 cache are those of paged_attn_split.cu; what differs is
// the bound: with 256 rows a key costs 4 * 256 * head_dim operations, so the products run on tcgen05 and the softmax beside them.
//
// One CTA per SM takes a block of 256 rows (two halves of 128) through tiles of 128 keys:
//   warps 0-3, 4-7   softmax of half 0 and 1, a thread per row (= TMEM lane): no shuffles.  They also load the rows of q at the
//                    start of a block and write the output at its end.
//   warps 8-11       loaders: keys and values into a ring of [128 keys][D] 16-bit slots, 128-byte swizzle, K(0) V(0) K(1) V(1) ...
//                    Both caches go by cp.async, a bf16 one into the slot, an E4M3 one into a staging area from which the thread that
//                    asked for the bytes converts them (exactly, to fp16).
//                    Keys that are not there are stored as zeros, so whatever lies in their place reaches no product.
//   warp 12          issues the products.  S_h = Q_h K^T (both from shared memory) into TMEM; the softmax turns S_h into P_h (fp16 or
//                    bf16) over the same TMEM columns; O_h += P_h V with P_h as the tensor-memory operand and V as it lies, rows of
//                    D contiguous elements (MN-major).  The order PV_0(j) S_0(j+1) PV_1(j) S_1(j+1) keeps the tensor cores on one half while
//                    the other half's softmax runs.
// A block of no more than 128 rows has no second half: its even tiles go through S_0, O_0 and warps 0-3, its odd tiles through S_1, O_1
// and warps 4-7, with a running maximum and sum of their own, and warps 0-3 join the two at the end (the same TMEM lanes hold the
// same rows).  With one half alone the block was one chain of product, softmax, product (24 sequences of up to 16 new on up to 8192 tokens, 32/4
// heads of 64: 49 us, 45 us so).
// TMEM: S_0 S_1 (128 columns each), O_0 O_1 (D columns each).  The running maximum is raised, and O rescaled in TMEM by the row's
// own thread, only when it grows by more than 2^4 (exact: the sum uses the same base); after the first tiles that is rare.
#include "paged_common.cuh"
#include "paged_attn.cuh"
#include "ptx.cuh"

namespace b200q {
namespace paged {
namespace chunk {

constexpr int kRows = 256, kTile = 128, kThreads = 512;
constexpr int kScaleSlots = 4;
constexpr int kSoftmaxRegs = 200, kLoaderRegs = 72, kMmaRegs = 40;            // 2 * 200 + 72 + 40 = 4 * 128
// The exponents of a tile's value scales, from smallest to largest, up to which the row's n is taken from the largest of them and of its
// scores: it is then 2^kSpread too high at most, so an operand keeps its bits down to 2^-(25 - kSpread) of the row's largest.  A tile
// of wider spread is walked twice, key by key.
constexpr uint32_t kSpread = 12;
// Power of two, either way, up to which a tile's value scales are not far from one: where all have been so, n - m is as near to 0 as
// they are (and kLazy more), and 2^(x - n) serves for the row's sum as well.
constexpr uint32_t kNear = 56;

template <int D, bool FP8>
struct Cfg {
    static constexpr int kHalves = D / 64;                                    // 128-byte columns of a 16-bit row
    static constexpr int kHalfBytes = kTile * 128;
    static constexpr int kSlotBytes = kHalves * kHalfBytes;
    static constexpr int kSlots = D == 64 ? 6 : FP8 ? 3 : 4;
    static constexpr int kStagedBytes = FP8 ? kTile * D : 0;                  // E4M3 bytes of a tile of keys or values, on their way
    static constexpr int kStaged = D == 64 ? 6 : 3;
    static constexpr int kQBytes = 2 * kSlotBytes;
    // per tile: mask words, largest and smallest exponent fields of the value scales, words of the keys whose value scale is not
    // finite (4 each), key scales, value scales
    static constexpr int kScaleAt = 64;
    static constexpr int kScaleBytes = kScaleAt + (FP8 ? 2 * kTile * 4 : 0);
    static constexpr int kBars = 2 * kSlots + kScaleSlots + 12;
    static constexpr int kSmemBytes = 1024 + kQBytes + kSlots * kSlotBytes + kStaged * kStagedBytes + kScaleSlots * kScaleBytes + kBars * 8 + 64 + 128 * 16;
    static constexpr int kOCol = 256;
    static_assert(kQBytes + kSlots * kSlotBytes >= 8192 * 4, "a word per sequence");
};

// 16-byte unit `unit` of row `row` in a [rows][128 bytes] column with the 128-byte swizzle
__device__ __forceinline__ uint32_t unit_at(uint32_t column, int row, int unit) { return column + row * 128 + ((unit ^ (row & 7)) << 4); }

// Keys first .. first + 31 that the position of a row lets it see, as bits.
__device__ __forceinline__ uint32_t visible_keys(int causal, int window, int pos, int first)
{
    const int last = causal ? pos - first : 31, from = window > 0 ? pos - window + 1 - first : 0;
    const uint32_t upto = last < 0 ? 0u : last >= 31 ? 0xFFFFFFFFu : (2u << last) - 1u;
    return from <= 0 ? upto : from > 31 ? 0u : upto & ~((1u << from) - 1u);
}

// A row's accumulators times f; the products so far are done.
template <int D>
__device__ __forceinline__ void rescale_output(uint32_t t_o, float f)
{
    ptx::tcgen05_fence_after_sync();
#pragma unroll 1
    for (int i = 0; i < D; i += 16) {
        uint32_t o[16];
        ptx::tmem_ld_32x32b_x16(t_o + i, o);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
        ptx::tmem_st_32x32b_x16(t_o + i, o);
    }
}

// P of 64 keys is on its way to tensor memory: once it is there, the products over them can start.
__device__ __forceinline__ void operands_stored(uint32_t bar)
{
    ptx::tmem_st_wait();
    ptx::tcgen05_fence_before_sync();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bar);
}

// The softmax of a tile of an E4M3 cache whose value scales are of wide spread, or far from one: walked twice through tensor memory, 32 keys at
// a time, with an exponential of its own for the sum and for the operand.  (A kernel without this branch takes 1178 us for the prefill chunks
// that take 1200 with it, inside the loop or, as here, out of line.)
struct Row {
    float m, n, l;
    bool ok;
};
template <int D>
__device__ __noinline__ Row tile_by_key(Row row, uint32_t t_s, uint32_t t_o, uint32_t key_scales, uint32_t masks, float row_scale, int causal, int window,
                                        int pos, int key0, bool fresh, uint32_t o_bar, uint32_t o_parity, uint32_t p_bar, uint32_t* status)
{
    auto scores = [&](int w, float (&x)[32]) {
        ptx::tmem_ld_32x32b_x32(t_s + 32 * w, reinterpret_cast<uint32_t (&)[32]>(x));
        ptx::tmem_ld_wait();
        const uint32_t seen = __float_as_uint(ptx::ld_shared_f32(masks + 4 * w)) & visible_keys(causal, window, pos, key0 + 32 * w);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            x[i] = x[i] * ptx::ld_shared_f32(key_scales + 4 * (32 * w + i)) * row_scale;
            if (!((seen >> i) & 1u)) x[i] = -INFINITY;
        }
    };
    auto value_scale = [&](int key) { return ptx::ld_shared_f32(key_scales + 4 * (kTile + key)); };
    float mn = row.m, nn = -INFINITY;
#pragma unroll 1
    for (int w = 0; w < 4; ++w) {
        float x[32];
        scores(w, x);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            mn = fmaxf(mn, x[i]);
            nn = fmaxf(nn, x[i] + log2_above(field_of(value_scale(32 * w + i))));
        }
    }
    const float om = mn == -INFINITY ? 0.0f : mn;
    row.l *= ptx::ex2(row.m - om);
    row.m = mn;
    float f = 1.0f;
    if (nn > row.n + kLazy) {
        f = ptx::ex2(row.n - nn);
        row.n = nn;
    }
    if (!fresh && __any_sync(0xffffffffu, f != 1.0f)) {
        row.ok = __all_sync(0xffffffffu, ptx::mbar_wait(o_bar, o_parity, status, 3));
        rescale_output<D>(t_o, f);
    }
    const float base = kRoomLog2 - (row.n == -INFINITY ? 0.0f : row.n);
#pragma unroll 1
    for (int w = 0; w < 4; ++w) {                                             // (P of 32 keys lies where the scores of 16 were)
        float x[32];
        uint32_t p[16];
        scores(w, x);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            float y[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float v = value_scale(32 * w + i + k);
                row.l += ptx::ex2(x[i + k] - om);
                y[k] = ptx::ex2(x[i + k] + (log2_above(field_of(v)) + base)) * mantissa_of(v);
            }
            p[i / 2] = pack_f16x2(y[0], y[1]);
        }
        ptx::tmem_st_32x32b_x16(t_s + 16 * w, p);
        if (w & 1) operands_stored(p_bar + 8u * (w >> 1));
    }
    return row;
}

template <int D, bool FP8>
__global__ void __launch_bounds__(kThreads, 1)
attn_chunk_kernel(const Args a)
{
    using C = Cfg<D, FP8>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = ptx::smem_u32(smem_raw);
    const uint32_t q_base = (raw + 1023u) & ~1023u;
    const uint32_t ring = q_base + C::kQBytes;
    const uint32_t staging = ring + C::kSlots * C::kSlotBytes;
    const uint32_t scales = staging + C::kStaged * C::kStagedBytes;
    const uint32_t bars = scales + kScaleSlots * C::kScaleBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };                     // a slot holds its tile
    auto empty_bar = [&](int s) { return bars + 8u * (C::kSlots + s); };
    auto scale_bar = [&](int s) { return bars + 8u * (2 * C::kSlots + s); };  // the softmax is done with a tile's scales
    const uint32_t more = bars + 8u * (2 * C::kSlots + kScaleSlots);
    auto q_bar = [&](int h) { return more + 8u * h; };
    auto s_bar = [&](int h) { return more + 8u * (2 + h); };                  // scores of half h are in TMEM
    auto p_bar = [&](int h, int k) { return more + 8u * (4 + 2 * h + k); };   // P of half h, keys 64 * k .., is in TMEM
    auto o_bar = [&](int h) { return more + 8u * (8 + h); };                  // P V of half h is done
    const uint32_t joined_bar = more + 8u * 10, read_bar = more + 8u * 11;    // odd tiles' states are there / have been read
    const uint32_t tmem_slot = bars + C::kBars * 8;
    int* block_info = reinterpret_cast<int*>(smem_raw + (tmem_slot + 4 - raw));        // for the products: tiles (0: no more blocks), halves
    float4* odd_state = reinterpret_cast<float4*>(smem_raw + ((bars + C::kBars * 8 + 48 + 15) / 16 * 16 - raw));       // [128] maximum, sum, poison
    int* odd_block = block_info + 3;                                          // [8] by the block's number: it has values that are not finite
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Shape& s = a.s;

    ptx::pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kSlots; ++i) { ptx::mbar_init(full_bar(i), FP8 ? 4 : 128); ptx::mbar_init(empty_bar(i), 1); }
        for (int i = 0; i < kScaleSlots; ++i) ptx::mbar_init(scale_bar(i), 8);
        for (int i = 0; i < 8; ++i) odd_block[i] = 0;
        for (int h = 0; h < 2; ++h) { ptx::mbar_init(q_bar(h), 4); ptx::mbar_init(s_bar(h), 1); ptx::mbar_init(p_bar(h, 0), 4); ptx::mbar_init(p_bar(h, 1), 4); ptx::mbar_init(o_bar(h), 1); }
        ptx::mbar_init(joined_bar, 4); ptx::mbar_init(read_bar, 4);
        ptx::fence_mbar_init();
        a.open[blockIdx.x].last = -1;
    }
    if (warp == 12) { ptx::tmem_alloc(tmem_slot, 512); ptx::tmem_relinquish(); }
    ptx::tcgen05_fence_before_sync();
    Cursor c = find_work(s, kRows, kTile, reinterpret_cast<int*>(smem_raw + (q_base - raw)), a.block_limit, a.block_most, blockIdx.x, gridDim.x);
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_raw + (tmem_slot - raw));
    Seq q{};
    if (c.at < c.end) q = load_seq(s, c.b);
    bool ok = true;
    // Whether some row of a block does not see a key of the tile that others do.  Values there that are not finite (in a bf16 cache) would
    // pass the product as 0 * infinity into the rows that do not see them: the loaders set them to zero, note it for the
    // block, and the rows that do see them get them at the end.
    auto edge = [&](const Range& r, int i, int tile) {
        const int first = max(tile * kTile, r.lo), end = min(tile * kTile + kTile, r.hi);
        const int r1 = min(q.n * s.group, (i + 1) * kRows) - 1;
        return first < end && ((s.causal && end - 1 > q.kv - q.n + s.token_of(i * kRows)) ||
                               (s.window > 0 && first <= q.kv - q.n + s.token_of(r1) - s.window));
    };
    int block_no = 0;                                                         // blocks so far, the same in all roles

    if (warp < 8) {
        // ================================================================================================ softmax
        ptx::regs_inc<kSoftmaxRegs>();
        const int h = warp >> 2, quad = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t t_s = tmem + lanes + h * 128, t_o = tmem + lanes + C::kOCol + h * D;
        uint32_t s_phase = 0, o_phase = 0, join_phase = 0;
        int slot = 0;                                                         // of the scale ring
        while (c.at < c.end && ok) {
            ++block_no;
            const Range r = block_range(s, q, c.i, kRows, kTile);
            const int todo = min(r.tiles - c.tile, c.end - c.at);
            const int r0 = c.i * kRows, rows = min(kRows, q.n * s.group - r0);
            const bool two = rows > 128;                                      // two halves of rows; else odd tiles go to h = 1
            const int r_in = (two ? h * 128 : 0) + quad * 32 + lane;          // row inside the block
            const bool half_on = two || todo > h, warp_on = (two ? h * 128 : 0) + quad * 32 < rows;
            const int row = min(r_in, rows - 1);                              // rows behind the block repeat its last one
            const int tok = s.token_of(r0 + row), head = c.h * s.group + (r0 + row) - tok * s.group;
            const int pos = q.kv - q.n + tok;
            const size_t out_row = static_cast<size_t>(q.q0 + tok) * s.heads + head;
            float row_scale = fabsf(a.scale_log2);
            if (half_on) {
                // ---- the warp's rows of q into shared memory, a few whole rows at a time (code that runs once a block is bound by
                // the fetch of its instructions: short loops, not unrolled ones); the sign of the softmax scale goes into them,
                // so that the factor of the scores is not negative (nor zero)
                const long long q_row = (q.q0 + tok) * a.q_stride + head * a.q_head;
                const float sign = a.scale_log2 > 0.0f ? 1.0f : a.scale_log2 < 0.0f ? -1.0f : 0.0f;
                if (a.scale_log2 == 0.0f) row_scale = 1.0f;
                constexpr int kLanes = D / 8, kAt = 32 / kLanes;              // lanes of a row, rows at a time
                const int piece = lane % kLanes, sub = lane / kLanes;
                uint32_t my_e = 127;
#pragma unroll 8
                for (int i = 0; i < 32 / kAt; ++i) {
                    const int rr = i * kAt + sub;
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(a.q + __shfl_sync(0xffffffffu, q_row, rr)) + piece);
                    float down = sign;
                    if (FP8) {
                        uint32_t m2 = __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
                        uint32_t mx = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
                        for (int o = 1; o < kLanes; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        const uint32_t e = min(max(mx >> 7, 1u), 253u);       // exponent field of the row's largest element
                        down *= pow2_of_field(254u - e);
                        const uint32_t mine = __shfl_sync(0xffffffffu, e, (lane % kAt) * kLanes);
                        if (lane / kAt == i) my_e = mine;
                    }
                    uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float lo = __uint_as_float(v[k] << 16) * down, hi = __uint_as_float(v[k] & 0xFFFF0000u) * down;
                        v[k] = FP8 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
                    }
                    if (two || h == 0) ptx::st_shared_v4(unit_at(q_base + h * C::kSlotBytes + (piece >> 3) * C::kHalfBytes, quad * 32 + rr, piece & 7), v[0], v[1], v[2], v[3]);
                }
                // (not zero, which would make a hidden key's -infinity NaN: tiny rows times a tiny softmax scale)
                if (FP8) row_scale = fmaxf(row_scale * pow2_of_field(my_e), __uint_as_float(1u));
                ptx::fence_proxy_async_smem();
                if (threadIdx.x == 0) { block_info[0] = todo; block_info[1] = two ? 2 : 1; }
                __syncwarp();
                if (lane == 0 && (two || h == 0)) ptx::mbar_arrive(q_bar(h));
            }
            const int pos_lo = __shfl_sync(0xffffffffu, pos, 0), pos_hi = __shfl_sync(0xffffffffu, pos, 31);
            // m, n: the bases of the row's sum and of its operands (paged_common.cuh)
            float m = -INFINITY, n = -INFINITY, l = 0.0f, poison = 0.0f;
            bool fresh = true;                                                // O holds nothing of this block yet
            bool far = false;                                                 // some row of the warp has n far from m
            for (int t = 0; t < todo && ok; ++t) {
                const uint32_t sc = scales + slot * C::kScaleBytes;
                const bool mine = two || (t & 1) == h;
                if (mine) {
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait(s_bar(h), s_phase, a.status, 2));
                    if (!ok) break;
                    s_phase ^= 1u;
                    ptx::tcgen05_fence_after_sync();
                    if (warp_on) {
                        const int key0 = (r.tile0 + c.tile + t) * kTile;
                        const uint4 mask = ptx::ld_shared_v4(sc);
                        auto visible = [&](int w) { return visible_keys(s.causal, s.window, pos, key0 + 32 * w); };
                        // O of the tiles so far, on a new base
                        auto rescale = [&](float f) {
                            if (fresh || !__any_sync(0xffffffffu, f != 1.0f)) return;
                            ok = __all_sync(0xffffffffu, ptx::mbar_wait(o_bar(h), o_phase ^ 1u, a.status, 3));
                            rescale_output<D>(t_o, f);
                        };
                        uint32_t v_top = 0;                                   // exponent field of the largest value scale
                        bool by_key = false;
                        if (FP8) {
                            const uint4 odd = ptx::ld_shared_v4(sc + 48), top4 = ptx::ld_shared_v4(sc + 16), low4 = ptx::ld_shared_v4(sc + 32);
                            v_top = max(max(top4.x, top4.y), max(top4.z, top4.w));
                            const uint32_t v_low = min(min(low4.x, low4.y), min(low4.z, low4.w));
                            by_key = v_top > v_low + kSpread || v_top - (127u - kNear) > 2 * kNear || far;
                            if ((odd.x | odd.y | odd.z | odd.w) != 0u &&
                                ((odd.x & visible(0)) | (odd.y & visible(1)) | (odd.z & visible(2)) | (odd.w & visible(3))) != 0u)
                                poison = __uint_as_float(0x7FC00000u);
                        }
                        if (FP8 && __builtin_expect(by_key, 0)) {
                            // value scales of wide spread, or far from one
                            const Row to = tile_by_key<D>(Row{m, n, l, ok}, t_s, t_o, sc + C::kScaleAt, sc, row_scale, s.causal, s.window, pos, key0, fresh,
                                                          o_bar(h), o_phase ^ 1u, p_bar(h, 0), a.status);
                            m = to.m; n = to.n; l = to.l; ok = to.ok;
                            far = __any_sync(0xffffffffu, fabsf(n - m) > kNear + 2 * kLazy);
                        } else {
                            float x[kTile];
#pragma unroll
                            for (int i = 0; i < 4; ++i) ptx::tmem_ld_32x32b_x32(t_s + 32 * i, reinterpret_cast<uint32_t (&)[32]>(x[32 * i]));
                            ptx::tmem_ld_wait();
                            if (FP8) {
#pragma unroll
                                for (int i = 0; i < kTile; i += 4) {
                                    const uint4 k4 = ptx::ld_shared_v4(sc + C::kScaleAt + 4 * i);
                                    const float2 u = ptx::mul2(make_float2(x[i], x[i + 1]), make_float2(__uint_as_float(k4.x), __uint_as_float(k4.y)));
                                    const float2 v = ptx::mul2(make_float2(x[i + 2], x[i + 3]), make_float2(__uint_as_float(k4.z), __uint_as_float(k4.w)));
                                    x[i] = u.x; x[i + 1] = u.y; x[i + 2] = v.x; x[i + 3] = v.y;
                                }
                            }
                            const bool whole = (mask.x & mask.y & mask.z & mask.w) == 0xFFFFFFFFu && (!s.causal || key0 + kTile - 1 <= pos_lo) &&
                                               (s.window == 0 || key0 > pos_hi - s.window);
                            if (!whole) {
                                const uint32_t mk[4] = {mask.x, mask.y, mask.z, mask.w};
#pragma unroll
                                for (int w = 0; w < 4; ++w) {
                                    const uint32_t seen = mk[w] & visible(w);
#pragma unroll
                                    for (int i = 0; i < 32; ++i)
                                        if (!((seen >> i) & 1u)) x[32 * w + i] = -INFINITY;
                                }
                            }
                            float mx[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                            for (int i = 4; i < kTile - 4; i += 8)
#pragma unroll
                                for (int k = 0; k < 4; ++k) mx[k] = ptx::max3(mx[k], x[i + k], x[i + 4 + k]);
#pragma unroll
                            for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], x[kTile - 4 + k]);
                            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * row_scale;
                            float f = 1.0f;
                            if (top > m + kLazy || m == -INFINITY) {
                                const float mn = fmaxf(m, top);
                                f = ptx::ex2(m - (mn == -INFINITY ? 0.0f : mn));
                                m = mn;
                            }
                            l *= f;
                            if (FP8) {
                                // (the keys' own scales are at most 2^kSpread below the largest)
                                const float nn = top + log2_above(v_top);
                                const bool up = nn > n + kLazy;
                                f = up ? ptx::ex2(n - nn) : 1.0f;
                                if (up) n = nn;
                            }
                            rescale(f);
                            // E4M3: 2^kRoomLog2 2^(x - n), for the operand and, times 2^(n - m), for the sum: n - m is small in this branch
                            const float om = m == -INFINITY ? 0.0f : m, on = n == -INFINITY ? 0.0f : n, base = FP8 ? kRoomLog2 - on : -om;
                            const float2 rs2 = make_float2(row_scale, row_scale), b2 = make_float2(base, base);
                            float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                            for (int g = 0; g < kTile; g += 64) {
                                uint32_t p[32];
#pragma unroll
                                for (int i = 0; i < 64; i += 4) {
                                    float2 u = ptx::fma2(make_float2(x[g + i], x[g + i + 1]), rs2, b2);
                                    float2 v = ptx::fma2(make_float2(x[g + i + 2], x[g + i + 3]), rs2, b2);
                                    u = make_float2(ptx::ex2(u.x), ptx::ex2(u.y));
                                    v = make_float2(ptx::ex2(v.x), ptx::ex2(v.y));
                                    sum[0] = ptx::add2(sum[0], u);
                                    sum[1] = ptx::add2(sum[1], v);
                                    if (FP8) {
                                        const uint4 y = ptx::ld_shared_v4(sc + C::kScaleAt + 4 * kTile + 4 * (g + i));
                                        u = ptx::mul2(u, make_float2(__uint_as_float(y.x), __uint_as_float(y.y)));
                                        v = ptx::mul2(v, make_float2(__uint_as_float(y.z), __uint_as_float(y.w)));
                                        p[i / 2] = pack_f16x2(u.x, u.y);
                                        p[i / 2 + 1] = pack_f16x2(v.x, v.y);
                                    } else {
                                        p[i / 2] = pack_bf16x2(u.x, u.y);
                                        p[i / 2 + 1] = pack_bf16x2(v.x, v.y);
                                    }
                                }
                                ptx::tmem_st_32x32b_x32(t_s + g / 2, p);
                                operands_stored(p_bar(h, g / 64));
                            }
                            sum[0] = ptx::add2(sum[0], sum[1]);
                            l += (sum[0].x + sum[0].y) * (FP8 ? ptx::ex2(on - om - kRoomLog2) : 1.0f);
                        }
                    } else if (lane == 0) {
                        ptx::mbar_arrive(p_bar(h, 0));
                        ptx::mbar_arrive(p_bar(h, 1));
                    }
                    o_phase ^= 1u;                                            // the tile's P V completes one more phase
                    fresh = false;
                }
                // eight arrivals a tile: one of each warp, or two of each that has the tile to itself
                __syncwarp();
                if (lane == 0 && mine) {
                    ptx::mbar_arrive(scale_bar(slot));
                    if (!two) ptx::mbar_arrive(scale_bar(slot));
                }
                if (++slot == kScaleSlots) slot = 0;
            }
            if (half_on && ok) {
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(o_bar(h), o_phase ^ 1u, a.status, 3));
                ptx::tcgen05_fence_after_sync();
                const bool begins = c.tile == 0, ends = c.tile + todo == r.tiles;
                const int part = 2 * blockIdx.x + (begins ? 1 : 0);
                float* po = a.part + static_cast<size_t>(part) * kRows * (D + 2);
                const bool whole_block = begins && ends, joins = !two && todo > 1;
                const float own = FP8 ? n : m;                                // what O stands on
                float to1 = -INFINITY;                                        // ... of the odd tiles, where they are joined
                if (joins && h == 1) {
                    odd_state[quad * 32 + lane] = make_float4(m, l, poison, own);
                    ptx::tcgen05_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(joined_bar);
                    ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(read_bar, join_phase, a.status, 8));
                } else if (joins) {
                    ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait(joined_bar, join_phase, a.status, 8));
                    ptx::tcgen05_fence_after_sync();
                    const float4 st = odd_state[quad * 32 + lane];
                    const float mn = fmaxf(m, st.x), base = mn == -INFINITY ? 0.0f : mn;
                    l = l * ptx::ex2(m - base) + st.y * ptx::ex2(st.x - base);
                    m = mn;
                    to1 = st.w;
                    poison += st.z;
                }
                if (joins) join_phase ^= 1u;
                const float inv = !whole_block ? 1.0f : l == 0.0f ? 0.0f : __frcp_rn(l);
                // O of this half and of the other on the common base; E4M3: in two steps, since 2^(n - m) alone may lie outside the
                // range of the numbers
                const float base = m == -INFINITY ? 0.0f : m;
                float f0 = 1.0f, f1 = 0.0f, g0 = 1.0f, g1 = 0.0f;
                if (FP8) {
                    g0 = ptx::ex2(0.5f * (own - base));
                    g1 = ptx::ex2(0.5f * (to1 - base));
                    f0 = g0 * (inv * kRoomInv);
                    f1 = g1 * (inv * kRoomInv);
                } else {
                    f0 = (joins ? ptx::ex2(own - base) : 1.0f) * inv;
                    f1 = ptx::ex2(to1 - base) * inv;
                }
                if (warp_on && (two || h == 0)) {
                    // A thread has a row: written from here, every 16 bytes would be a line of their own.  The rows of q (whose products
                    // are done) lend the warp their place in shared memory, 256 (D = 64: 128) bytes a row, and it writes whole rows.
                    const uint32_t place = q_base + h * C::kSlotBytes;
                    const int my = quad * 32 + lane, in_warp = min(32, rows - (r_in - lane));
                    constexpr int kPieces = D / 8;                            // 16-byte pieces of a row's place
                    auto flush = [&](int col, bool f32) {
                        __syncwarp();
#pragma unroll 2
                        for (int i = 0; i < kPieces; ++i) {                   // 32 * kPieces pieces, 32 at a time
                            const int rr = i * (32 / kPieces) + lane / kPieces, piece = lane % kPieces;
                            const uint4 w = ptx::ld_shared_v4(unit_at(place + (piece >> 3) * C::kHalfBytes, quad * 32 + rr, piece & 7));
                            const size_t to = __shfl_sync(0xffffffffu, out_row, rr);
                            if (rr < in_warp) {
                                if (f32) *reinterpret_cast<uint4*>(po + (r_in - lane + rr) * D + col + piece * 4) = w;
                                else *reinterpret_cast<uint4*>(a.out + to * D + piece * 8) = w;
                            }
                        }
                        __syncwarp();
                    };
#pragma unroll 1
                    for (int i = 0; i < D; i += 32) {
                        uint32_t o[32];
                        ptx::tmem_ld_32x32b_x32(t_o + i, o);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * (FP8 ? g0 : 1.0f) * f0 + poison);
                        if (joins) {
                            uint32_t y[32];
                            ptx::tmem_ld_32x32b_x32(t_o + D + i, y);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(y[k]) * (FP8 ? g1 : 1.0f) * f1 + __uint_as_float(o[k]));
                        }
                        if (!FP8 && *static_cast<volatile int*>(odd_block + (block_no & 7)) == block_no) {
#pragma unroll 1
                            for (int key = (r.tile0 + c.tile) * kTile; key < (r.tile0 + c.tile + todo) * kTile; ++key) {
                                if (key < r.lo || key >= r.hi || !edge(r, c.i, key / kTile)) continue;
                                const int page = __ldg(s.table + static_cast<size_t>(c.b) * s.max_pages + (key >> s.page_shift));
                                if (page < 0 || page >= s.num_pages) continue;
                                const size_t from = (static_cast<size_t>(page * s.kv_heads + c.h) << s.page_shift) + (key & ((1 << s.page_shift) - 1));
                                const bool seen = (!s.causal || key <= pos) && (s.window == 0 || key > pos - s.window);
#pragma unroll
                                for (int k = 0; k < 32; k += 2) {
                                    const uint32_t w = __ldg(static_cast<const uint32_t*>(a.v_cache) + (from * D + i + k) / 2);
                                    const uint32_t odd = w ^ only_finite(w);
                                    if (seen && (odd & 0xFFFFu)) o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(w << 16));
                                    if (seen && (odd >> 16)) o[k + 1] = __float_as_uint(__uint_as_float(o[k + 1]) + __uint_as_float(w & 0xFFFF0000u));
                                }
                            }
                        }
                        if (whole_block) {
#pragma unroll
                            for (int k = 0; k < 32; k += 8) {
                                uint32_t w[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(__uint_as_float(o[k + 2 * e]), __uint_as_float(o[k + 2 * e + 1]));
                                const int unit = (i + k) / 8;
                                ptx::st_shared_v4(unit_at(place + (unit >> 3) * C::kHalfBytes, my, unit & 7), w[0], w[1], w[2], w[3]);
                            }
                        } else {
                            // 32 columns are half (D = 64: all) of the place
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                const int unit = (i % (D / 2) + k) / 4;
                                ptx::st_shared_v4(unit_at(place + (unit >> 3) * C::kHalfBytes, my, unit & 7), o[k], o[k + 1], o[k + 2], o[k + 3]);
                            }
                            if ((i + 32) % (D / 2) == 0) flush(i + 32 - D / 2, true);
                        }
                    }
                    if (whole_block) flush(0, false);
                    if (r_in < rows) {
                        if (!whole_block) *reinterpret_cast<float2*>(po + kRows * D + r_in * 2) = make_float2(m, l);
                        else if (a.lse != nullptr) a.lse[out_row] = lse_of(m, l);
                    }
                }
                ptx::tcgen05_fence_before_sync();
                if (joins && h == 0) {
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(read_bar);
                }
                if (threadIdx.x == 0 && begins && !ends) {
                    Open* op = a.open + blockIdx.x;
                    op->token0 = q.q0; op->r0 = r0; op->rows = rows; op->h = c.h;
                    op->last = owner(c, c.at + r.tiles - 1);
                }
            }
            c.at += todo;
            if (c.at < c.end) next_block(s, c, q, kRows);
        }
        if (h == 0 && ok) {
            if (threadIdx.x == 0) block_info[0] = 0;
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(q_bar(0));
        }
    } else if (warp < 12) {
        // ================================================================================================ loaders
        ptx::regs_dec<kLoaderRegs>();
        const int lw = warp - 8;                                              // keys 32 * lw .. + 31 of a tile
        int slot = 0, sslot = 0;
        uint32_t phase = 0, sphase = 0;
        int stage_in = 0, stage_out = 0;                                      // E4M3: of the staging area's items
        while (c.at < c.end && ok) {
            ++block_no;
            const Range r = block_range(s, q, c.i, kRows, kTile);
            const int todo = min(r.tiles - c.tile, c.end - c.at);
            const int* table = s.table + static_cast<size_t>(c.b) * s.max_pages;
            // the cache row of this lane's key of a tile, -1 for none
            auto row_of = [&](int tile) {
                const int key = tile * kTile + lw * 32 + lane;
                if (key < r.lo || key >= r.hi) return -1;
                const int page = __ldg(table + (key >> s.page_shift));
                if (page < 0 || page >= s.num_pages) return -1;
                return ((page * s.kv_heads + c.h) << s.page_shift) + (key & ((1 << s.page_shift) - 1));
            };
            constexpr int kPerRow = (FP8 ? D : 2 * D) / 16;                   // 16-byte pieces of a row
            constexpr int kRowsAt = 32 / kPerRow;                             // rows a warp instruction covers
            constexpr int kInstr = 32 / kRowsAt;                              // instructions of a warp's 32 rows
            // E4M3 rows of 128: eight neighbouring lanes take four pieces of two rows, so that their stores of 32 bytes hit eight
            // different 16-byte units
            const int piece = FP8 && D == 128 ? (lane & 3) + ((lane >> 1) & 4) : lane % kPerRow;
            const int sub = FP8 && D == 128 ? ((lane >> 2) & 1) + ((lane >> 3) & 2) : lane / kPerRow;
            // E4M3: a thread's pieces wait in its own places of the staging area until it converts them
            const uint32_t staged = staging + (lw * 32 + lane) * 16;
            uint32_t at[8 / kRowsAt > 0 ? 8 / kRowsAt : 1][2];                // where a piece's 16 elements (two units) go; the swizzle repeats after 8 rows
            if constexpr (FP8) {
#pragma unroll
                for (int o = 0; o < 8 / kRowsAt; ++o)
#pragma unroll
                    for (int u = 0; u < 2; ++u) at[o][u] = unit_at((piece >> 2) * C::kHalfBytes, lw * 32 + o * kRowsAt + sub, (piece & 3) * 2 + u);
            }
            auto stage_item = [&](const void* cache, int rows_of_lane) {
                const uint32_t to = staged + stage_in * C::kStagedBytes;
#pragma unroll
                for (int i = 0; i < kInstr; ++i) {
                    const int from = __shfl_sync(0xffffffffu, rows_of_lane, i * kRowsAt + sub);
                    ptx::cp_async_16(to + i * 2048, static_cast<const uint8_t*>(cache) + static_cast<size_t>(max(from, 0)) * D + piece * 16, from >= 0 ? 16u : 0u);
                }
                ptx::cp_async_commit();
                if (++stage_in == C::kStaged) stage_in = 0;
            };
            // items are staged kStaged - 1 ahead (one tile, or two and a half); scales one tile ahead; rows as far as the items need them
            constexpr int kFar = C::kStaged / 2;                              // tiles between an item and the one staged with it
            int rows_ahead[kFar + 1];
#pragma unroll
            for (int i = 0; i <= kFar; ++i) rows_ahead[i] = i < todo ? row_of(r.tile0 + c.tile + i) : -1;
            float ks = 0.0f, vs = 0.0f;
            if (FP8) {
                if (rows_ahead[0] >= 0) { ks = __ldg(a.k_scale + rows_ahead[0]); vs = __ldg(a.v_scale + rows_ahead[0]); }
#pragma unroll
                for (int i = 0; i < C::kStaged - 1; ++i) stage_item(i % 2 == 0 ? a.k_cache : a.v_cache, rows_ahead[i / 2]);
            }
            for (int t = 0; t < todo && ok; ++t) {
                const int row = rows_ahead[0];
                const int after = t + kFar + 1 < todo ? row_of(r.tile0 + c.tile + t + kFar + 1) : -1;
                float ks_next = 0.0f, vs_next = 0.0f;
                if (FP8 && rows_ahead[1] >= 0) { ks_next = __ldg(a.k_scale + rows_ahead[1]); vs_next = __ldg(a.v_scale + rows_ahead[1]); }
                // ---- the tile's mask and scales
                ok = __all_sync(0xffffffffu, ptx::mbar_wait(scale_bar(sslot), sphase ^ 1u, a.status, 4));
                if (!ok) break;
                {
                    const uint32_t sc = scales + sslot * C::kScaleBytes;
                    uint8_t* scp = smem_raw + (sc - raw);
                    const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
                    const uint32_t bits = __float_as_uint(vs) & 0x7FFFFFFFu;
                    const uint32_t odd = __ballot_sync(0xffffffffu, bits >= 0x7F800000u);
                    // (a scale that is not finite reaches its rows by itself; one below the smallest normal number counts as zero)
                    const uint32_t field = bits >= 0x7F800000u ? 0u : bits >> 23;
                    if (field == 0u) vs = 0.0f;
                    const uint32_t top = __reduce_max_sync(0xffffffffu, field), low = __reduce_min_sync(0xffffffffu, field == 0u ? 255u : field);
                    if (lane == 0) {
                        reinterpret_cast<uint32_t*>(scp)[lw] = there;
                        reinterpret_cast<uint32_t*>(scp)[4 + lw] = top;
                        reinterpret_cast<uint32_t*>(scp)[8 + lw] = low;
                        reinterpret_cast<uint32_t*>(scp)[12 + lw] = odd;
                    }
                    if (FP8) {
                        reinterpret_cast<float*>(scp + C::kScaleAt)[lw * 32 + lane] = ks;
                        reinterpret_cast<float*>(scp + C::kScaleAt)[kTile + lw * 32 + lane] = vs;
                    }
                    if (++sslot == kScaleSlots) { sslot = 0; sphase ^= 1u; }
                }
                // ---- keys, then values
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    const uint8_t* cache = static_cast<const uint8_t*>(kv == 0 ? a.k_cache : a.v_cache);
                    if (FP8) {
                        // the item kStaged - 1 further on: with an odd distance of the other kind
                        constexpr bool kOther = (C::kStaged - 1) % 2 != 0;
                        const int far = kOther && kv == 1 ? rows_ahead[kFar] : rows_ahead[(C::kStaged - 1) / 2];
                        stage_item(kOther == (kv == 0) ? a.v_cache : a.k_cache, far);   // (empty items behind the last tile)
                        ptx::cp_async_wait<C::kStaged - 1>();
                    }
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait(empty_bar(slot), phase ^ 1u, a.status, 1));
                    if (!ok) break;
                    const uint32_t to = ring + slot * C::kSlotBytes;
                    if constexpr (FP8) {
                        const uint32_t from = staged + stage_out * C::kStagedBytes;
#pragma unroll
                        for (int i = 0; i < kInstr; ++i) {
                            const uint4 w = ptx::ld_shared_v4(from + i * 2048);
                            constexpr int kPeriod = 8 / kRowsAt;
                            const uint32_t go = to + (i / kPeriod) * 1024;
                            ptx::st_shared_v4(go + at[i % kPeriod][0], ptx::e4m3x2_lo(w.x), ptx::e4m3x2_hi(w.x), ptx::e4m3x2_lo(w.y), ptx::e4m3x2_hi(w.y));
                            ptx::st_shared_v4(go + at[i % kPeriod][1], ptx::e4m3x2_lo(w.z), ptx::e4m3x2_hi(w.z), ptx::e4m3x2_lo(w.w), ptx::e4m3x2_hi(w.w));
                        }
                        if (++stage_out == C::kStaged) stage_out = 0;
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive(full_bar(slot));
                    } else {
#pragma unroll
                        for (int i = 0; i < kInstr; ++i) {
                            const int from = __shfl_sync(0xffffffffu, row, i * kRowsAt + sub);
                            ptx::cp_async_16(unit_at(to + (piece >> 3) * C::kHalfBytes, lw * 32 + i * kRowsAt + sub, piece & 7),
                                             cache + static_cast<size_t>(max(from, 0)) * (2 * D) + piece * 16, from >= 0 ? 16u : 0u);
                        }
                        if (kv == 1 && edge(r, c.i, r.tile0 + c.tile + t)) {
                            ptx::cp_async_commit();
                            ptx::cp_async_wait<0>();
#pragma unroll 2
                            for (int i = 0; i < kInstr; ++i) {                // each thread looks at what it copied
                                const uint32_t at_piece = unit_at(to + (piece >> 3) * C::kHalfBytes, lw * 32 + i * kRowsAt + sub, piece & 7);
                                const uint4 y = ptx::ld_shared_v4(at_piece);
                                const uint4 z = make_uint4(only_finite(y.x), only_finite(y.y), only_finite(y.z), only_finite(y.w));
                                if (((y.x ^ z.x) | (y.y ^ z.y) | (y.z ^ z.z) | (y.w ^ z.w)) != 0u) {
                                    ptx::st_shared_v4(at_piece, z.x, z.y, z.z, z.w);
                                    odd_block[block_no & 7] = block_no;
                                }
                            }
                            ptx::fence_proxy_async_smem();
                            ptx::mbar_arrive(full_bar(slot));                 // (every thread is one of the barrier's arrivals)
                        } else {
                            ptx::cp_async_arrive(full_bar(slot));             // as many items in flight as there are slots
                        }
                    }
                    if (++slot == C::kSlots) { slot = 0; phase ^= 1u; }
                }
#pragma unroll
                for (int i = 0; i < kFar; ++i) rows_ahead[i] = rows_ahead[i + 1];
                rows_ahead[kFar] = after;
                ks = ks_next; vs = vs_next;
            }
            if (FP8) {
                ptx::cp_async_wait<0>();                                      // the empty items
                stage_in = stage_out;
            }
            c.at += todo;
            if (c.at < c.end) next_block(s, c, q, kRows);
        }
        if (!FP8) {
            ptx::cp_async_commit();
            ptx::cp_async_wait<0>();
        }
    } else {
        // ================================================================================================ products
        ptx::regs_dec<kMmaRegs>();
        if (warp == 12 && ptx::elect_one()) {
            constexpr uint32_t fmt = FP8 ? 0u : 1u;                           // fp16 / bf16
            constexpr uint32_t id_s = ptx::umma_idesc(fmt, fmt, 128, kTile);
            constexpr uint32_t id_o = ptx::umma_idesc(fmt, fmt, 128, D) | ptx::kIdescBMnMajor;
            int slot = 0;
            uint32_t phase = 0, q_phase[2] = {0, 0}, p_phase[2] = {0, 0};
            // copied (not converted) tiles reach the barrier by the copies themselves: their writers pass no proxy fence
            auto landed = [&]() { if (!FP8) ptx::fence_proxy_async_smem(); };
            auto advance = [&]() { if (++slot == C::kSlots) { slot = 0; phase ^= 1u; } };
            auto scores = [&](int h, int q_half, uint32_t k_at) {
                const uint64_t dq = ptx::smem_desc_sw128_kmajor(q_base + q_half * C::kSlotBytes), dk = ptx::smem_desc_sw128_kmajor(k_at);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint64_t step = (i >> 2) * (C::kHalfBytes >> 4) + 2 * (i & 3);
                    ptx::umma_f16(tmem + h * 128, dq + step, dk + step, id_s, i > 0);
                }
                ptx::umma_commit(s_bar(h));
            };
            while (ok) {
                // scores of the first tile
                ok = ptx::mbar_wait(q_bar(0), q_phase[0], a.status, 6);
                if (!ok) break;
                q_phase[0] ^= 1u;
                const int todo = *static_cast<volatile int*>(block_info), halves = *static_cast<volatile int*>(block_info + 1);
                if (todo == 0) break;
                ok = ptx::mbar_wait(full_bar(slot), phase, a.status, 5);
                for (int h = 0; h < halves && ok; ++h) {
                    if (h == 1) {
                        ok = ptx::mbar_wait(q_bar(1), q_phase[1], a.status, 6);
                        q_phase[1] ^= 1u;
                    }
                    ptx::tcgen05_fence_after_sync();
                    landed();
                    if (ok) scores(h, h, ring + slot * C::kSlotBytes);
                }
                ptx::umma_commit(empty_bar(slot));
                advance();
                for (int t = 0; t < todo && ok; ++t) {
                    const int v_slot = slot;
                    const uint32_t v_phase = phase;
                    advance();
                    const bool on = t + 1 < todo;
                    const int k_slot = slot;
                    const uint32_t k_phase = phase;
                    if (on) advance();
                    if (halves == 1 && on) {                                  // the next tile's scores go to the other S first
                        ok = ptx::mbar_wait(full_bar(k_slot), k_phase, a.status, 5);
                        if (!ok) break;
                        ptx::tcgen05_fence_after_sync();
                        landed();
                        scores((t + 1) & 1, 0, ring + k_slot * C::kSlotBytes);
                        ptx::umma_commit(empty_bar(k_slot));
                    }
                    for (int n = 0; n < halves && ok; ++n) {
                        const int h = halves == 2 ? n : t & 1;
                        const bool sum = halves == 2 ? t > 0 : t > 1;         // O_h holds earlier tiles
                        if (n == 0) { ok = ptx::mbar_wait(full_bar(v_slot), v_phase, a.status, 5); landed(); }
                        const uint64_t dv = ptx::smem_desc_sw128_mnmajor(ring + v_slot * C::kSlotBytes, C::kHalfBytes);
#pragma unroll
                        for (int i = 0; i < kTile / 16; ++i) {                // 16 keys: 8 columns of P, 2 KB of each column of V
                            if (i % 4 == 0) {
                                ok = ok && ptx::mbar_wait(p_bar(h, i / 4), p_phase[h], a.status, 7);
                                if (!ok) break;
                                ptx::tcgen05_fence_after_sync();
                            }
                            ptx::umma_f16_ts(tmem + C::kOCol + h * D, tmem + h * 128 + 8 * i, dv + (2048 >> 4) * i, id_o, sum || i > 0);
                        }
                        if (!ok) break;
                        p_phase[h] ^= 1u;
                        ptx::umma_commit(o_bar(h));
                        if (n == halves - 1) ptx::umma_commit(empty_bar(v_slot));
                        if (halves == 2 && on) {
                            if (n == 0) {
                                ok = ptx::mbar_wait(full_bar(k_slot), k_phase, a.status, 5);
                                if (!ok) break;
                                ptx::tcgen05_fence_after_sync();
                                landed();
                            }
                            scores(h, h, ring + k_slot * C::kSlotBytes);
                            if (n == 1) ptx::umma_commit(empty_bar(k_slot));
                        }
                    }
                }
            }
        }
        __syncwarp();
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 12) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc(tmem, 512);
    }
}

template <int D, bool FP8>
int launch(const Args& args, cudaStream_t stream)
{
    using C = Cfg<D, FP8>;
    Args a = args;
    auto kernel = attn_chunk_kernel<D, FP8>;
    static bool configured[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
        if (e != cudaSuccess) return e;
        if (dev < 64) configured[dev] = true;
    }
    if (!tiles_fit(a, kRows, kTile)) return cudaErrorInvalidValue;
    a.block_limit = static_cast<int>((static_cast<long long>(a.max_q) * a.s.group + kRows - 1) / kRows);
    a.block_most = static_cast<int>(most_blocks(a, kRows));          // (tiles_fit bounds it)
    const int ctas = num_sms();
    kernel<<<ctas, kThreads, C::kSmemBytes, stream>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_combine<D>(a, ctas, kRows, stream);
}

}  // namespace chunk

int attn_chunk(const Args& a, int head_dim, bool fp8, cudaStream_t stream)
{
    if (head_dim == 64) return fp8 ? chunk::launch<64, true>(a, stream) : chunk::launch<64, false>(a, stream);
    return fp8 ? chunk::launch<128, true>(a, stream) : chunk::launch<128, false>(a, stream);
}

size_t attn_chunk_part_bytes(int head_dim) { return static_cast<size_t>(num_sms()) * 2 * chunk::kRows * (head_dim + 2) * sizeof(float); }

}  // namespace paged
}  // namespace b200q
