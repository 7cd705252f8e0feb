// Entry point of the attention over a paged cache: argument checks and the choice of kernel.
#include "paged_attn.cuh"
#include "../../include/b200q.h"

namespace b200q {
namespace paged {
int page_shift_of(int page_size);        // paged_cache.cu
// Rows per kv head up to which the split-KV kernel is taken.  It reads the keys once per 16 rows, mostly from L2; the tensor-core kernel
// once, but takes longer to start.  24 sequences of up to 8192 tokens, heads 32/4 of 64, bf16: 38 / 47 / 61 / 74 us with 16 / 32 / 48 / 64
// rows against 53 us; heads 5/5, E4M3, 42 rows: 36 / 37; heads 8/8 of 128, E4M3, 44 rows: 40 / 41; heads 4/1, 52 rows: 46 / 52.
constexpr int kSplitRows = 48;
// ... and pairs of a block of 16 rows and a tile of 64 keys up to which it is taken whatever the rows are (counted from the sizes
// of the call, so an upper bound).  Heads 32/8 of 128, E4M3, split-KV against tensor cores: one sequence, 64 new on 512 (1024 pairs)
// 18 / 32 us, 128 on 512 (2048) 24 / 33, 64 on 2048 (4096) 32 / 34, 256 on 1024 (8192) 52 / 37; 64 sequences, 32 on 64 (2408) 42 / 38.
// A window bounds the tiles a block sees: one sequence, 21 new on 4587, window 429, heads 40/5 of 64, bf16: 13.1 / 23.2.
constexpr long long kSplitPairs = 4096;
bool few_pairs(const Args& a)
{
    long long tiles = ((static_cast<long long>(a.s.max_pages) << a.s.page_shift) + 63) / 64;
    if (a.s.window > 0) {                            // the 16 rows are at most 16 / group + 1 tokens, rounded up
        const long long seen = (static_cast<long long>(a.s.window) + (15 + a.s.group) / a.s.group + 62) / 64 + 1;
        tiles = seen < tiles ? seen : tiles;
    }
    return most_blocks(a, 16) * tiles <= kSplitPairs;
}
int g_impl = 0;                          // 0 by the number of rows, 1 split-KV kernel, 2 tensor-core kernel
size_t open_bytes() { return (static_cast<size_t>(attn_split_ctas()) * sizeof(Open) + 15) / 16 * 16; }
}
}

extern "C" {

size_t b200q_paged_attention_workspace_bytes(int head_dim)
{
    if (head_dim != 64 && head_dim != 128) return 0;
    const size_t split = b200q::paged::attn_split_part_bytes(head_dim), chunk = b200q::paged::attn_chunk_part_bytes(head_dim);
    return b200q::paged::open_bytes() + (split > chunk ? split : chunk);
}

int b200q_paged_attention(const void* q, const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                          const int* page_table, const int* cu_q, const int* kv_lens, void* out, float* lse, int seqs, int tokens,
                          int heads, int kv_heads, int head_dim, long long q_stride, long long q_head_stride, int max_q, int max_pages,
                          int num_pages, int page_size, int fp8, float softmax_scale, int causal, int window, int zero_rest,
                          void* workspace, void* stream)
{
    using namespace b200q;
    using namespace b200q::paged;
    if (q == nullptr || k_cache == nullptr || v_cache == nullptr || page_table == nullptr || cu_q == nullptr || kv_lens == nullptr ||
        out == nullptr || workspace == nullptr) return cudaErrorInvalidValue;
    if (fp8 && (k_scale == nullptr || v_scale == nullptr)) return cudaErrorInvalidValue;
    const int shift = page_shift_of(page_size);
    if (seqs <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || max_q <= 0 || max_pages <= 0 ||
        num_pages <= 0 || shift < 0 || (head_dim != 64 && head_dim != 128)) return cudaErrorInvalidValue;
    if (window < 0 || (window > 0 && !causal) || !(softmax_scale == softmax_scale)) return cudaErrorInvalidValue;
    if (q_stride % 8 || q_head_stride % 8 || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(out) ||
        !aligned16(workspace) || (fp8 && (!aligned16(k_scale) || !aligned16(v_scale)))) return cudaErrorInvalidValue;
    // the work is counted in shared memory, a word per sequence
    if (seqs > 8192) return cudaErrorInvalidValue;
    // positions, rows of a chunk and rows of the cache are 32-bit numbers
    const long long most = 0x7FFFFFFFll - 4096;
    if ((static_cast<long long>(max_pages) << shift) > most || static_cast<long long>(tokens) * heads > most ||
        ((static_cast<long long>(num_pages) * kv_heads) << shift) > most) return cudaErrorInvalidValue;
    if (num_sms() <= 0) return cudaErrorInvalidDevice;

    Args a{};
    a.s.cu_q = cu_q; a.s.kv_lens = kv_lens; a.s.table = page_table;
    a.s.seqs = seqs; a.s.tokens = tokens; a.s.heads = heads; a.s.kv_heads = kv_heads; a.s.set_group(heads / kv_heads);
    a.s.max_pages = max_pages; a.s.page_shift = shift; a.s.num_pages = num_pages;
    a.s.causal = causal != 0; a.s.window = window;
    a.q = static_cast<const __nv_bfloat16*>(q); a.q_stride = q_stride; a.q_head = q_head_stride;
    a.k_cache = k_cache; a.v_cache = v_cache; a.k_scale = k_scale; a.v_scale = v_scale;
    a.out = static_cast<__nv_bfloat16*>(out); a.lse = lse;
    a.scale_log2 = softmax_scale * 1.44269504088896341f;
    a.max_q = max_q < tokens ? max_q : tokens;
    a.zero_rest = zero_rest != 0;
    a.status = status_ptr();
    if (a.status == nullptr) return cudaErrorInvalidDevice;
    a.open = static_cast<Open*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + open_bytes());
    const bool chunk = g_impl != 0 ? g_impl == 2 : static_cast<long long>(a.max_q) * a.s.group > kSplitRows && !few_pairs(a);
    return chunk ? attn_chunk(a, head_dim, fp8 != 0, static_cast<cudaStream_t>(stream)) : attn_split(a, head_dim, fp8 != 0, static_cast<cudaStream_t>(stream));
}

int b200q_paged_set_impl(int impl)
{
    if (impl < 0 || impl > 2) return cudaErrorInvalidValue;
    b200q::paged::g_impl = impl;
    return 0;
}

}  // extern "C"
