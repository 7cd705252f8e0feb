// What the paged-cache operators share: the shape of a call, which keys a block of query rows sees, and how a persistent
// grid divides the work of a ragged batch.
//
// Cache layout: [pages, kv_heads, page_size, head_dim] for keys and for values (bf16, or E4M3 bytes with one fp32 scale per
// row in [pages, kv_heads, page_size]): the tokens of one page and head are one contiguous run, so a tile of keys is a few
// boxes of a 2-D tensor map over rows, and a row is (page * kv_heads + head) * page_size + offset.
#pragma once
#include "common.cuh"

namespace b200q {
namespace paged {

// One call of the attention.  The rows of a sequence's chunk of n tokens are ordered (token, head of the group), row
// r = token * group + g, for each kv head: query heads that share keys share a tile.
struct Shape {
    const int* cu_q;          // [seqs + 1] first row of each sequence's chunk in q
    const int* kv_lens;       // [seqs] cached tokens, the chunk included
    const int* table;         // [seqs, max_pages]
    int seqs, tokens, heads, kv_heads, group;
    int max_pages, page_shift, num_pages;
    int causal, window;       // window 0 = none; a window implies causal
    unsigned group_mul, group_shift;        // x / group without a division: see token_of

    // Token of row r of a chunk, r / group, for 0 <= r < 2^31: with s = ceil(log2 group) and mul = ceil(2^(31 + s) / group) the
    // product r * mul / 2^(31 + s) is off by less than 1 / group (mul * group exceeds 2^(31 + s) by less than 2^s), so its
    // integer part is the quotient.  A row's code runs once per block and is bound by instruction fetch, where a division
    // costs twenty of them.
    __host__ void set_group(int g)
    {
        group = g;
        group_shift = 0;
        while ((1 << group_shift) < g) ++group_shift;
        group_mul = static_cast<unsigned>(((1ull << (31 + group_shift)) + g - 1) / g);
    }
    __host__ __device__ int token_of(int r) const
    {
        return static_cast<int>((static_cast<unsigned long long>(r) * group_mul) >> (31 + group_shift));
    }
};

// Lengths as the caller gave them, made safe: whatever the arrays hold, rows stay inside q and keys inside the table.
struct Seq {
    int q0, n, kv, cap;
};
__device__ __forceinline__ Seq load_seq(const Shape& s, int b)
{
    Seq q;
    q.q0 = min(max(__ldg(s.cu_q + b), 0), s.tokens);
    q.n = min(max(__ldg(s.cu_q + b + 1), q.q0), s.tokens) - q.q0;
    q.kv = max(__ldg(s.kv_lens + b), 0);
    q.cap = min(q.kv, s.max_pages << s.page_shift);
    return q;
}

// Keys [lo, hi) that some row of block i (rows i * rm .. of the chunk) sees, and the tiles of kt keys that hold them.  A block
// that sees nothing gets one empty tile: its rows are written (as zero) like any others.
struct Range {
    int lo, hi, tile0, tiles;
};
__device__ __forceinline__ Range block_range(const Shape& s, const Seq& q, int i, int rm, int kt)
{
    const int r0 = i * rm, r1 = min(q.n * s.group, r0 + rm);
    const int first = q.kv - q.n + s.token_of(r0), last = q.kv - q.n + s.token_of(r1 - 1);   // positions of the block's tokens
    Range r;
    r.hi = s.causal ? min(q.cap, last + 1) : q.cap;
    r.lo = s.window > 0 && first >= s.window ? first - s.window + 1 : 0;       // (a negative position less a large window would pass 32 bits)
    if (r.lo >= r.hi) { r.lo = 0; r.hi = 0; }
    r.tile0 = r.lo / kt;
    r.tiles = max(1, (r.hi + kt - 1) / kt - r.tile0);
    return r;
}

// The work of a call is the list of all tiles: sequence by sequence, kv head by kv head, row block by row block, tile by
// tile.  The CTAs take equal shares of it (of kMinTiles at least), whatever the lengths are; a long sequence is split over as
// many CTAs as it takes.  A block whose tiles lie in several CTAs leaves partial results (running maximum, sum,
// unnormalised output), joined by the combine kernel in CTA order.  Tile counts are 32-bit numbers: the host refuses calls whose
// sizes could pass that, and starts that contradict one another (chunks that overlap) and pass it all the same do no work.
// Tiles a CTA has at least: a part costs a write, a read and a turn of the combine kernel (one sequence of 1500 tokens, 8 kv heads: 13.9 us with
// 1, 11.5 with 2, 11.3 with 3, 11.7 with 4).  But as many CTAs as there are blocks, where the grid has them: a block costs its CTA more
// than a tile does (one token on 36, heads 32/8 of 128: 11.4 us with three blocks a CTA, 6.5 with one; 40 sequences, up to 4 new on
// 130: 22.5 and 17.0; tensor-core kernel, one token on 36: 24 and 11.7).
constexpr int kMinTiles = 3;
struct Cursor {
    int b, h, i;              // sequence, kv head, row block
    int tile;                 // first tile (counted from the block's tile0) this CTA takes of the block
    int at, end;              // this CTA's tiles, as indices of the list; at == end: nothing left
    int share, extra;         // tiles of a CTA; the first `extra` CTAs have one more
};

constexpr int kTooMany = 0x7FFFFFFF;
__device__ __forceinline__ int add_capped(int a, int b)           // a, b in [0, kTooMany]
{
    return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), static_cast<unsigned>(kTooMany)));
}
__device__ __forceinline__ int capped(long long w) { return static_cast<int>(min(w, static_cast<long long>(kTooMany))); }

// Whole CTA; `prefix` holds seqs words in shared memory (free again after the call, which ends in a barrier).
// `block_limit`: an upper bound of the row blocks of one sequence, `block_most`: of all blocks (row blocks times kv heads).
__device__ __forceinline__ Cursor find_work(const Shape& s, int rm, int kt, int* prefix, int block_limit, int block_most, int cta, int ctas)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (block_limit <= 8) {                        // a thread per sequence
        for (int b = threadIdx.x; b < s.seqs; b += blockDim.x) {
            const Seq q = load_seq(s, b);
            const int blocks = (q.n * s.group + rm - 1) / rm;
            long long w = 0;
            for (int i = 0; i < blocks; ++i) w += block_range(s, q, i, rm, kt).tiles;
            prefix[b] = capped(w * s.kv_heads);
        }
    } else {                                       // a warp per sequence
        for (int b = warp; b < s.seqs; b += warps) {
            const Seq q = load_seq(s, b);
            const int blocks = (q.n * s.group + rm - 1) / rm;
            long long w = 0;
            for (int i = lane; i < blocks; i += 32) w += block_range(s, q, i, rm, kt).tiles;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
            if (lane == 0) prefix[b] = capped(w * s.kv_heads);
        }
    }
    __syncthreads();
    if (warp == 0) {                               // inclusive prefix sums
        int run = 0;
        for (int b0 = 0; b0 < s.seqs; b0 += 32) {
            int v = b0 + lane < s.seqs ? prefix[b0 + lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v = add_capped(v, u);
            }
            v = add_capped(v, run);
            if (b0 + lane < s.seqs) prefix[b0 + lane] = v;
            run = __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
    const int counted = s.seqs > 0 ? prefix[s.seqs - 1] : 0, total = counted == kTooMany ? 0 : counted;
    const int used = min(ctas, max((total + kMinTiles - 1) / kMinTiles, min(total, block_most)));
    Cursor c{};
    if (cta < used) {
        c.share = total / used;
        c.extra = total - c.share * used;
        c.at = cta * c.share + min(cta, c.extra);
        c.end = c.at + c.share + (cta < c.extra ? 1 : 0);
        int lo = 0, hi = s.seqs - 1;               // first sequence whose inclusive prefix exceeds c.at
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (prefix[mid] > c.at) hi = mid; else lo = mid + 1;
        }
        c.b = lo;
        const int before = lo > 0 ? prefix[lo - 1] : 0;
        const int per_head = (prefix[lo] - before) / s.kv_heads;
        int rem = c.at - before;
        c.h = rem / per_head;
        rem -= c.h * per_head;
        const Seq q = load_seq(s, lo);
        for (c.i = 0;; ++c.i) {
            const int t = block_range(s, q, c.i, rm, kt).tiles;
            if (rem < t) break;
            rem -= t;
        }
        c.tile = rem;
    }
    __syncthreads();
    return c;
}

// The CTA that does tile t of the list.
__device__ __forceinline__ int owner(const Cursor& c, int t)
{
    const int head = c.extra * (c.share + 1);      // tiles of the CTAs that have one more
    return t < head ? t / (c.share + 1) : c.extra + (t - head) / c.share;
}

// The next block after (b, h, i), called while tiles are left; sequences without rows are passed over.
__device__ __forceinline__ void next_block(const Shape& s, Cursor& c, Seq& q, int rm)
{
    c.tile = 0;
    if ((c.i + 1) * rm < q.n * s.group) { ++c.i; return; }
    c.i = 0;
    if (++c.h < s.kv_heads) return;
    c.h = 0;
    do { q = load_seq(s, ++c.b); } while (q.n == 0);
}

// What a CTA leaves for the combine kernel: the block whose first tiles it did and whose last it did not.
struct Open {
    int token0;               // first row of the sequence's chunk in q
    int r0, rows, h;          // the block
    int last;                 // CTA that does the block's last tile; -1: nothing open
};

// E4M3 cache: the second product takes p_j s_j (s_j the scale of value j) in fp16.  Each row keeps two running maxima, both in units of
// log2: m of its scores x_j, on which its sum of 2^(x_j - m) stands, and n of x_j + e_j with 2^e_j the power of two above s_j, on which
// its operands and its accumulators stand: the product's operand is 2^(x_j - n) s_j 2^kRoomLog2.  So what fp16 keeps depends on what the row itself uses
// of its values, not on the scales of keys that it does not see, has left behind or gives no weight.  n is raised only when
// it grows by more than kLazy, so an operand is below 2^(kRoomLog2 + kLazy) = 2^15; it loses bits where it is below 2^-14, that is
// 2^-25 of n's key.  Scales below the smallest normal number (the write makes none) count as zero.
constexpr int kRoomLog2 = 11;
constexpr float kRoomInv = 1.0f / 2048.0f;
constexpr float kLazy = 4.0f;
__device__ __forceinline__ float pow2_of_field(uint32_t e) { return __uint_as_float(e << 23); }      // 2^(e - 127), 1 <= e <= 254
__device__ __forceinline__ uint32_t field_of(float x) { return (__float_as_uint(x) >> 23) & 255u; }
__device__ __forceinline__ float log2_above(uint32_t field) { return static_cast<float>(static_cast<int>(field) - 126); }   // e_j
// s / 2^e_j: 0.5 to 1 in magnitude, 0 for a zero; infinities and NaN as they are
__device__ __forceinline__ float mantissa_of(float s)
{
    const uint32_t b = __float_as_uint(s), f = field_of(s);
    return f == 255u ? s : f == 0u ? 0.0f : __uint_as_float((b & 0x807FFFFFu) | 0x3F000000u);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// two bf16 with those that are not finite set to zero
__device__ __forceinline__ uint32_t only_finite(uint32_t w)
{
    if ((w & 0x7F80u) == 0x7F80u) w &= 0xFFFF0000u;
    if ((w & 0x7F800000u) == 0x7F800000u) w &= 0x0000FFFFu;
    return w;
}

}  // namespace paged
}  // namespace b200q
