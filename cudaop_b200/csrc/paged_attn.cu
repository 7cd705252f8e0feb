// Entry point of the attention over a paged cache: argument checks and the choice of kernel.
#include "paged_attn.cuh"
#include "../../include/b200q.h"

namespace b200q {
namespace paged {
int page_shift_of(int page_size);        // paged_cache.cu
// Which kernel.  The split-KV kernel reads the keys once per 16 rows, mostly from L2; the tensor-core kernel once, but takes longer to start.
// Figures are split-KV / tensor cores in us; chunks of equal length on the given lengths, 8 kv heads of 128, 32 heads unless said.
//
// E4M3 cache (p has 11 bits in both).  Up to 32 rows per kv head the split-KV kernel: 64 sequences of 1024 tokens, 16 / 24 / 32 / 40 / 48 rows:
// 62/118, 106/120, 108/121, 153/120, 156/120; 256 of 256: 89/170, 155/180, 164/181, 232/183, 239/181; 24 of up to 8192, heads 32/4: 48/78,
// 91/88, 87/89, 103/70, 140/93.  With more rows where the call is small, counted in blocks of 16 rows and tiles of 64 keys from its sizes (an
// upper bound), a block costing about as much as eight tiles: one sequence, 64 new on 512 (2048) 20/33, 128 on 512 (4096) 26/34, 64 on
// 2048 (5120) 35/35, 128 on 1024 (6144) 41/39, 256 on 1024 (12288) 59/37; 8 sequences, 16 on 256 tokens 19/15; 64, 32 on 64 (36864) 88/39.
//
// bf16 cache.  The split-KV kernel holds p in two bf16 terms, the tensor-core kernel in one (8 bits), so it is kept for longer than its time alone
// would have it: 64 sequences of 1024 tokens, 32 / 40 / 48 rows: 119/104, 169/104, 170/105, heads of 64 68/68, 96/68, 97/68; 64 sequences, 32 on
// 64 (4096 pairs of a block and a tile): 79/37; one sequence, 128 on 1024 (4096): 36/34, 256 on 1024 (8192): 61/36.
constexpr int kSplitRowsE4m3 = 32, kSplitRowsBf16 = 48;
constexpr long long kSplitWork = 4096;
bool split_kernel(const Args& a, bool fp8)
{
    if (static_cast<long long>(a.max_q) * a.s.group <= (fp8 ? kSplitRowsE4m3 : kSplitRowsBf16)) return true;
    long long tiles = ((static_cast<long long>(a.s.max_pages) << a.s.page_shift) + 63) / 64;
    // A window bounds the tiles a block sees (one sequence, 21 new on 4587, window 429, heads 40/5 of 64, bf16: 13/23): the 16 rows are at
    // most 16 / group + 1 tokens, rounded up.
    if (a.s.window > 0) {
        const long long seen = (static_cast<long long>(a.s.window) + (15 + a.s.group) / a.s.group + 62) / 64 + 1;
        tiles = seen < tiles ? seen : tiles;
    }
    return most_blocks(a, 16) * (tiles + (fp8 ? 8 : 0)) <= kSplitWork;
}
int g_impl = 0;                          // 0 by the rule above, 1 split-KV kernel, 2 tensor-core kernel
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
    const bool split = g_impl != 0 ? g_impl == 1 : split_kernel(a, fp8 != 0);
    return split ? attn_split(a, head_dim, fp8 != 0, static_cast<cudaStream_t>(stream)) : attn_chunk(a, head_dim, fp8 != 0, static_cast<cudaStream_t>(stream));
}

int b200q_paged_set_impl(int impl)
{
    if (impl < 0 || impl > 2) return cudaErrorInvalidValue;
    b200q::paged::g_impl = impl;
    return 0;
}

}  // extern "C"
