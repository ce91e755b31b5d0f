/*
 * b200_kv4.h — a prefix K/V cache held in 4 bits, in pages: storing into it, joint
 * attention over it, reading it back, and moving its pages.
 *
 * The reference keeps each layer's prefix keys and values as one dense bf16 tensor
 * (TextKvCache, src/transformer.rs:14-45) and, when that does not fit, moves it to the
 * host (set_kv_cache_offload, 27-45).  Here it takes 144 bytes per token and head instead
 * of 512 and stays on the GPU; sequences with a common prefix share its pages.
 *
 * Pool of one layer: device uint8 [num_pages][heads][B200_KV4_BLOCK_BYTES], 16-byte
 * aligned.  A page holds 64 consecutive tokens of one sequence; page_table[b][i] is the
 * page of tokens [64 i, 64 i + 64) of batch row b.  Entries behind a row's last token are
 * not read.
 *
 * Values.  Each token's 128 channels form 4 groups of 32.  A group keeps one step s and 32
 * numbers n in [-7, 7]; the value is s * n.
 *   top = max |x| of the group;  s = top / 7 cut to 5 significant bits
 *   n = sign(x) * floor(|x| / s + 1/2)   (|x| / s < 7.44)
 *   top < 2^-100: s = 0, n = 0.  top >= 2^126 or not finite: s = NaN and n = 0, so that the
 *   whole group reads as NaN.
 * 5 bits of s times 3 bits of n: every value is exactly a bf16 number, so reading the cache
 * rounds nothing.
 *
 * Block of one head (bytes; a = token / 8 within the page, channel group c = channel / 32;
 * a nibble holds n + 8, low nibble first):
 *   [0, 4096)     K numbers: token 8a + g, channel 32c + 8t + j at nibble j of the 32-bit
 *                 word a*128 + (4g + t)*4 + c
 *   [4096, 8192)  V numbers: token 8a + 2t + p, channel 32c + 4g + i at nibble 4p + i of
 *                 the 32-bit word a*128 + (4g + t)*4 + c
 *   [8192, 8704)  K steps, bf16: token 8a + 2t + p, group c at element a*32 + t*8 + 2c + p
 *   [8704, 9216)  V steps, bf16: the same order
 * This is the order in which a warp's matrix fragments take them: lane 4g + t of a warp
 * reads 16 bytes, and the warp 512 bytes in a row.
 *
 * Conventions are those of b200_attn.h.  heads * head_dim of q, k and v equal the pool's:
 * one K/V head per query head.  status: optional device int32; B200_KV4_STATUS_BAD_PAGE is
 * left in it (if it was 0) when a page id outside [0, num_pages) or a position outside the
 * page table was met: such tokens are not stored, and read as zeros.
 */
#ifndef B200_KV4_H
#define B200_KV4_H

#include <stddef.h>
#include <stdint.h>

#include "b200_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_KV4_PAGE_TOKENS 64
#define B200_KV4_BLOCK_BYTES 9216
#define B200_KV4_STATUS_BAD_PAGE 16

/* One layer's pool and the page tables of a batch. */
typedef struct {
  void* pool;                /* device [num_pages][heads][B200_KV4_BLOCK_BYTES]          */
  const int32_t* page_table; /* device [batch][max_pages]                                */
  int32_t num_pages;         /* pages of the pool                                        */
  int32_t max_pages;         /* entries of one row of page_table                         */
} b200_kv4_view;

/*
 * Stores tokens [0, count[b]) of k and v at positions start[b] + i of batch row b's
 * sequence.  k, v: bf16, element (b, h, t, d) at b*sb + h*sh + t*st + d (strides in
 * elements, multiples of 8; the cache's post-RoPE keys, and values).  start, count: device
 * int32 [batch], or NULL (0 and `tokens`); count is limited to [0, tokens].  Bytes of other
 * tokens of a page are left as they are.  Two batch rows must not store into one page.
 * One kernel.
 */
int b200_kv4_store(const b200_kv4_view* cache, const void* k, int64_t k_sb, int64_t k_sh,
                   int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st,
                   int32_t batch, int32_t heads, int32_t tokens, int32_t head_dim,
                   const int32_t* start, const int32_t* count, int32_t* status,
                   b200_stream_t stream);

/*
 * Reads the cache back: k_out, v_out device bf16 [batch][heads][max_len][128], the dense
 * prefix layout of b200_attn_fwd; rows at and behind lengths[b * length_stride] are zeros.
 * lengths: device int32, limited to [0, max_len]; max_len <= 64 * max_pages.  One kernel.
 */
int b200_kv4_load(const b200_kv4_view* cache, const int32_t* lengths, int32_t length_stride,
                  void* k_out, void* v_out, int32_t batch, int32_t heads, int32_t max_len,
                  int32_t head_dim, int32_t* status, b200_stream_t stream);

/* Scratch bytes of b200_kv4_joint_attention for these sizes; 0 for few query rows (up to 64,
 * and up to 128 where batch * heads <= 64 and prefix_len >= 4 * target_len). */
int b200_kv4_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t target_len,
                                       int32_t prefix_len, size_t* bytes);

/*
 * b200_joint_attention with the prefix in this cache: q_rot, k_rot device [B,H,T,128], v
 * device [B,T,H,128], out device [B,T,H*128], all bf16 and dense.  Query row i of batch row
 * b attends to the cache's tokens [0, desc[b].prefix_valid) and to this call's keys
 * [0, desc[b].target_valid), of those only [0, row_limit[i]) where row_limit (device int32
 * [T], non-decreasing) is given.  prefix_len: a bound of every prefix_valid that the host
 * knows, <= 64 * max_pages; prefix_valid is limited to it.  desc NULL: prefix_len and T.
 * What k_rot and v hold behind target_valid, and the cache behind prefix_valid, does not
 * reach the output, infinities and NaN included.  A row without any key gives NaN (the
 * reference's softmax of a row of -inf), and so does a row that sees a key whose score is NaN
 * or +infinity (a stored group that was not finite reads as NaN).  An infinity or NaN in v of
 * a key that is valid but behind a row's row_limit may reach that row (0 * NaN is NaN, as in
 * a softmax times V).
 *
 * Few query rows run as one kernel straight from the 4-bit pages, without a workspace; for
 * more, the pages are expanded into the workspace once (b200_kv4_load's kernel) and the
 * tensor-core attention kernel reads them there.  Both work on the same values.  Calls that
 * may overlap need workspaces of their own.
 */
int b200_kv4_joint_attention(const b200_kv4_view* cache, const void* q_rot, const void* k_rot,
                             const void* v, int32_t batch, int32_t heads, int32_t target_len,
                             int32_t prefix_len, int32_t head_dim, const b200_kv_desc* desc,
                             const int32_t* row_limit, float scale, void* out, void* workspace,
                             size_t workspace_bytes, int32_t* status, b200_stream_t stream);

/*
 * b200_attn_fwd with the prefix in this cache: Q/K RMSNorm + RoPE, then
 * b200_kv4_joint_attention.  args as for b200_attn_fwd, with prefix_k and prefix_v NULL,
 * prefix_len the bound described above, and row_limit allowed with any prefix_len.
 */
int b200_kv4_attn_workspace_bytes(const b200_attn_args* args, size_t* bytes);
int b200_kv4_attn_fwd(const b200_attn_args* args, const b200_kv4_view* cache,
                      b200_stream_t stream);

/*
 * Copies whole pages within the pools of `layers` layers (layer l at pool + l *
 * layer_stride bytes): page dst[i] = page src[i], i < n.  src, dst: host arrays, read during
 * the call.  Refused (B200_ERR_INVALID): an id outside [0, num_pages), a page that is
 * written twice, and one that is both read and written (the copies run in no order).  One
 * kernel per 256 copies.
 */
int b200_kv4_copy_pages(void* pool, int32_t layers, int64_t layer_stride, int32_t num_pages,
                        int32_t heads, const int32_t* src, const int32_t* dst, int32_t n,
                        b200_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* B200_KV4_H */
