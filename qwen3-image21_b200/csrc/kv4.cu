// kv4.cu — the paged 4-bit prefix cache of include/b200_kv4.h: store, read back, page
// copies, and attention straight from the 4-bit pages for up to 64 query rows (128 of few
// heads); for more rows the pages are expanded for the attention of attn_fwd.cu.
//
//   kv4_store_kernel      one warp per 16 tokens of a page and head: group maxima by shuffles,
//                         numbers packed in registers, 16-byte stores in the block's order.
//                         4 x 4096 tokens of 32 heads: 60.6 us, 87 % of HBM's copy rate.
//   kv4_load_kernel       the inverse; s * n is exact in bf16.  The same tokens: 55.0 us, 95 %.
//   kv4_copy_kernel       16-byte copies of page pairs passed by value.  120 pages of 16
//                         layers: 174 us, 6.5 TB/s.
//   kv4_attn_kernel       up to 32 query rows, see there.
//   kv4_attn_tile_kernel  up to 64 (or 128), see there.
// The first three are bound by HBM (or, at a few pages, by their launch).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <vector>

#include "../../include/b200_kv4.h"
#include "attn_internal.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr int kHeadDim = 128;
constexpr int kPage = B200_KV4_PAGE_TOKENS;
constexpr int kBlock = B200_KV4_BLOCK_BYTES;
constexpr int kVOff = 4096;    // V numbers
constexpr int kKsOff = 8192;   // K steps
constexpr int kVsOff = 8704;   // V steps
constexpr int kOctetBytes = 512;      // numbers of 8 tokens
constexpr int kOctetStepBytes = 64;   // steps of 8 tokens
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
constexpr float kHuge = 8.507059173023462e37f;   // 2^126: 24 steps of a group stay finite

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  return __byte_perm(a, b, sel);
}

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

__device__ __forceinline__ void report_bad_page(int32_t* status) {
  if (status) atomicCAS(status, 0, B200_KV4_STATUS_BAD_PAGE);
}

// Nibbles i and i + 4 of w, each n + 8, as the bf16 pair 16 + u: u in the upper mantissa
// bits.  One three-input operation for the mask and the exponent (left to itself the
// compiler takes two, each with an immediate), and the shift to the left as a multiply,
// which keeps off the ALU pipe: that pipe bounds the expansion.
__device__ __forceinline__ uint32_t raw_pair(uint32_t w, int i) {
  const uint32_t at = i == 0 ? w * 8u : w >> (4 * i - 3);
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(at), "r"(0x00780078u), "r"(0x41804180u));
  return r;
}

// Nibbles i and i + 4 of w, each n + 8, times their steps: (16 + u) s - 24 s = n s in one packed
// fma.  The
// fma is exact: 24 s has at most 7 significant bits (s has 5) and n s has 8, so `less` =
// -24 s and the result are bf16 numbers.  A step of 0 gives 0, NaN gives NaN.
__device__ __forceinline__ uint32_t expand_pair(uint32_t w, int i, uint32_t step2, uint32_t less2) {
  const uint32_t v = raw_pair(w, i);
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                   *reinterpret_cast<const __nv_bfloat162*>(&step2),
                                   *reinterpret_cast<const __nv_bfloat162*>(&less2));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t less_of(uint32_t step2) {  // -24 s, exact
  const uint32_t k = 0xc1c0c1c0u;
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&step2),
                                   *reinterpret_cast<const __nv_bfloat162*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// ------------------------------------------------------------------ store
// The step of a group whose largest magnitude is `top` (a bf16 value, or NaN): top / 7 cut
// to 5 significant bits.  Cutting, not rounding: 7 s <= top, and top / s < 7.44 still has the
// number 7.  The factor is 1/7 rounded up by 2^-20: a quotient that is a 5-bit number does
// not fall below it, and any other is at least 1/7 unit of the 8-bit top away from one.
__device__ __forceinline__ float group_step(float top) {
  if (!(top < kHuge)) return __uint_as_float(0x7fc00000u);  // infinity, NaN, or too large
  if (top < kTiny) return 0.f;
  constexpr float kSeventh = static_cast<float>(1.0 / 7.0 * (1.0 + 0x1p-20));
  return __uint_as_float(__float_as_uint(top * kSeventh) & 0xfff80000u);
}

// The factor that number4 takes for a step above 0.
// |x| / s differs from a half by 0 or by at least 1/496 (x has 8 significant bits, s has 5,
// n at most 3): 1 + 2^-13 sends exact halves away from zero and moves no other value (below
// 7.44) across one.
__device__ __forceinline__ float number_scale(float step) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(step));
  return r * (1.f + 0x1p-13f);
}

// The numbers of a group, or 0 (8 in each nibble) for all of them where its step is 0 or NaN:
// taken by the step, not by a factor of 0, because infinity * 0 has no number.
__device__ __forceinline__ uint32_t numbers_of(float step, uint32_t numbers) {
  return step > 0.f ? numbers : 0x88888888u;
}

// n + 8 of the 4 values of two bf16 pairs as 4 nibbles in the low half: x * scale + 8 is
// rounded to an integer by adding 1.5 * 2^23, and the nibbles are put together in f32 (exact
// below 2^24), which keeps the work on the FMA pipe.
__device__ __forceinline__ uint32_t number4(uint32_t w0, uint32_t w1, float scale) {
  constexpr float kRound = 12582912.f;
  const float x[4] = {bf16_lo(w0), bf16_hi(w0), bf16_lo(w1), bf16_hi(w1)};
  float n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) n[i] = fmaf(x[i], scale, kRound + 8.f) - kRound;
  const float all = fmaf(n[3], 4096.f, fmaf(n[2], 256.f, fmaf(n[1], 16.f, n[0])));
  return __float_as_uint(all + 8388608.f);
}

// As bit patterns, magnitudes of bf16 values order like integers, with infinity above every
// finite value and NaN above infinity.
__device__ __forceinline__ uint32_t mag_max(uint32_t m, uint32_t pair) {
  return __vmaxu2(m, pair & 0x7fff7fffu);
}

struct StoreParams {
  uint8_t* pool;
  const int32_t* table;
  int32_t num_pages, max_pages;
  const __nv_bfloat16 *k, *v;
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  int32_t heads, tokens;
  const int32_t* start;
  const int32_t* count;
  int32_t* status;
};

// grid (page of the row's new tokens, head, batch row); warp w: tokens 16 w .. 16 w + 15 of
// the page.  Lane 4g + t holds, of K, token g's channels 32c + 8t + j and, of V, tokens
// 2t + {0, 1}, channels 32c + 4g + i — what the block wants of it as one 16-byte word per
// octet — so nothing is exchanged but the group maxima (over t for K, over g for V).  Global
// reads are 64-byte runs, stores 512-byte runs.
__global__ void __launch_bounds__(128, 6) kv4_store_kernel(const StoreParams p) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int64_t first = p.start ? p.start[b] : 0;
  const int64_t n = p.count ? min(max(p.count[b], 0), p.tokens) : p.tokens;
  // floor division: a negative start has its tokens before page 0
  const int64_t page_i = (first >= 0 ? first / kPage : -((-first + kPage - 1) / kPage)) + blockIdx.x;
  const int64_t base = page_i * kPage + warp * 16;  // position of this warp's first token
  if (base + 16 <= first || base >= first + n) return;
  int page = -1;  // looked at after the loads of k and v are on their way
  if (page_i >= 0 && page_i < p.max_pages) page = p.table[static_cast<int64_t>(b) * p.max_pages + page_i];
  const __nv_bfloat16* kb = p.k + b * p.k_sb + h * p.k_sh;
  const __nv_bfloat16* vb = p.v + b * p.v_sb + h * p.v_sh;
  const int64_t i0 = base - first;  // index of the warp's first token in k and v
  auto have = [&](int r) { return i0 + r >= 0 && i0 + r < n; };

  uint4 kx[2][4];      // [octet][group]: 8 channels
  uint2 vx[2][2][4];   // [octet][parity][group]: 4 channels
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int r = 8 * o + g;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      kx[o][c] = have(r) ? *reinterpret_cast<const uint4*>(kb + (i0 + r) * p.k_st + 32 * c + 8 * t)
                         : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int rv = 8 * o + 2 * t + q;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        vx[o][q][c] = have(rv) ? *reinterpret_cast<const uint2*>(vb + (i0 + rv) * p.v_st + 32 * c + 4 * g)
                               : make_uint2(0, 0);
    }
  }
  if (page < 0 || page >= p.num_pages) {
    if (lane == 0) report_bad_page(p.status);
    return;
  }
  uint8_t* block = p.pool + (static_cast<int64_t>(page) * p.heads + h) * kBlock;
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int octet = 2 * warp + o;
    // ---- K: two groups' maxima share a word in the shuffles
    uint32_t words[4];
    float step[4];
#pragma unroll
    for (int c = 0; c < 4; c += 2) {
      uint32_t m[2];
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint4 x = kx[o][c + z];
        m[z] = mag_max(mag_max(mag_max(mag_max(0u, x.x), x.y), x.z), x.w);
      }
      uint32_t both = __vmaxu2(prmt(m[0], m[1], 0x5410), prmt(m[0], m[1], 0x7632));
      both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, 1));
      both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, 2));
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint4 x = kx[o][c + z];
        step[c + z] = group_step(z ? bf16_hi(both) : bf16_lo(both));
        const float f = number_scale(step[c + z]);
        words[c + z] =
            numbers_of(step[c + z], prmt(number4(x.x, x.y, f), number4(x.z, x.w, f), 0x5410));
      }
    }
    if (have(8 * o + g)) {
      *reinterpret_cast<uint4*>(block + octet * kOctetBytes + lane * 16) =
          make_uint4(words[0], words[1], words[2], words[3]);
      // lane t writes group t's step of token g = 2t' + parity
      const float s = t == 0 ? step[0] : t == 1 ? step[1] : t == 2 ? step[2] : step[3];
      reinterpret_cast<uint16_t*>(block + kKsOff + octet * kOctetStepBytes)[(g >> 1) * 8 + 2 * t + (g & 1)] =
          static_cast<uint16_t>(__float_as_uint(s) >> 16);
    }
    // ---- V: the two tokens' maxima share a word
    uint32_t vw[4], vs[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint2 x0 = vx[o][0][c], x1 = vx[o][1][c];
      const uint32_t m0 = mag_max(mag_max(0u, x0.x), x0.y), m1 = mag_max(mag_max(0u, x1.x), x1.y);
      uint32_t both = __vmaxu2(prmt(m0, m1, 0x5410), prmt(m0, m1, 0x7632));
      both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, 4));
      both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, 8));
      both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, 16));
      const float s0 = group_step(bf16_lo(both)), s1 = group_step(bf16_hi(both));
      vs[c] = prmt(__float_as_uint(s0), __float_as_uint(s1), 0x7632);
      vw[c] = prmt(numbers_of(s0, number4(x0.x, x0.y, number_scale(s0))),
                   numbers_of(s1, number4(x1.x, x1.y, number_scale(s1))), 0x5410);
    }
    const bool h0 = have(8 * o + 2 * t), h1 = have(8 * o + 2 * t + 1);
    uint8_t* vd = block + kVOff + octet * kOctetBytes + lane * 16;
    uint8_t* sd = block + kVsOff + octet * kOctetStepBytes + t * 16;
    if (h0 && h1) {
      *reinterpret_cast<uint4*>(vd) = make_uint4(vw[0], vw[1], vw[2], vw[3]);
      if (g == 0) *reinterpret_cast<uint4*>(sd) = make_uint4(vs[0], vs[1], vs[2], vs[3]);
    } else if (h0 || h1) {  // one token of the pair: 16-bit stores leave the other's bytes
      const int q = h1 ? 1 : 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        reinterpret_cast<uint16_t*>(vd)[2 * c + q] = static_cast<uint16_t>(vw[c] >> (16 * q));
        if (g == 0) reinterpret_cast<uint16_t*>(sd)[2 * c + q] = static_cast<uint16_t>(vs[c] >> (16 * q));
      }
    }
  }
}

// ------------------------------------------------------------------ load
struct LoadParams {
  const uint8_t* pool;
  const int32_t* table;
  int32_t num_pages, max_pages;
  const int32_t* lengths;  // NULL: max_len
  int32_t length_stride;
  __nv_bfloat16 *k, *v;    // [B][H][max_len][128]
  int32_t heads, max_len;
  int32_t* status;
  int32_t* zero;  // n_zero words to clear for the launch behind this one, or NULL
  int32_t n_zero;
};

// grid (page, head, batch row), lanes as in the store.
__global__ void __launch_bounds__(128) kv4_load_kernel(const LoadParams p) {
  if (p.zero && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
    for (int i = threadIdx.x; i < p.n_zero; i += 128) p.zero[i] = 0;
  const int b = blockIdx.z, h = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int base = blockIdx.x * kPage + warp * 16;
  if (base >= p.max_len) return;
  const int len = p.lengths
                      ? min(max(p.lengths[static_cast<int64_t>(b) * p.length_stride], 0), p.max_len)
                      : p.max_len;
  const uint8_t* block = nullptr;
  if (base < len) {
    const int page = p.table[static_cast<int64_t>(b) * p.max_pages + blockIdx.x];
    if (page >= 0 && page < p.num_pages)
      block = p.pool + (static_cast<int64_t>(page) * p.heads + h) * kBlock;
    else if (lane == 0)
      report_bad_page(p.status);
  }
  const int64_t row0 = (static_cast<int64_t>(b) * p.heads + h) * p.max_len + base;
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int octet = 2 * warp + o;
    uint4 kw = make_uint4(0, 0, 0, 0), vw = kw, ks = kw, vs = kw;
    if (block) {
      kw = *reinterpret_cast<const uint4*>(block + octet * kOctetBytes + lane * 16);
      vw = *reinterpret_cast<const uint4*>(block + kVOff + octet * kOctetBytes + lane * 16);
      ks = *reinterpret_cast<const uint4*>(block + kKsOff + octet * kOctetStepBytes + (g >> 1) * 16);
      vs = *reinterpret_cast<const uint4*>(block + kVsOff + octet * kOctetStepBytes + t * 16);
    }
    const uint32_t kws[4] = {kw.x, kw.y, kw.z, kw.w}, vws[4] = {vw.x, vw.y, vw.z, vw.w};
    const uint32_t kss[4] = {ks.x, ks.y, ks.z, ks.w}, vss[4] = {vs.x, vs.y, vs.z, vs.w};
    const int rk = 8 * o + g;  // K: token g
    if (base + rk < p.max_len) {
      const bool live = block && base + rk < len;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t s2 = prmt(kss[c], kss[c], (g & 1) ? 0x3232 : 0x1010), less = less_of(s2);
        uint32_t pr[4];  // channels (i, i + 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = expand_pair(kws[c], i, s2, less);
        const uint4 out = make_uint4(prmt(pr[0], pr[1], 0x5410), prmt(pr[2], pr[3], 0x5410),
                                     prmt(pr[0], pr[1], 0x7632), prmt(pr[2], pr[3], 0x7632));
        *reinterpret_cast<uint4*>(p.k + (row0 + rk) * kHeadDim + 32 * c + 8 * t) =
            live ? out : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // V: tokens 2t, 2t + 1, pairs (token, token + 1)
      const uint32_t less = less_of(vss[c]);
      uint32_t pr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) pr[i] = expand_pair(vws[c], i, vss[c], less);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int rv = 8 * o + 2 * t + q;
        const uint32_t sel = q ? 0x7632 : 0x5410;
        if (base + rv < p.max_len)
          *reinterpret_cast<uint2*>(p.v + (row0 + rv) * kHeadDim + 32 * c + 4 * g) =
              block && base + rv < len ? make_uint2(prmt(pr[0], pr[1], sel), prmt(pr[2], pr[3], sel))
                                       : make_uint2(0, 0);
      }
    }
  }
}

// ------------------------------------------------------------------ page copies
constexpr int kPairs = 256;
constexpr int kCopyBytes = 16384;  // one CTA's part of a page

struct CopyParams {
  uint8_t* pool;
  int64_t layer_stride, page_bytes;
  int32_t src[kPairs], dst[kPairs];
};

__global__ void __launch_bounds__(256) kv4_copy_kernel(const __grid_constant__ CopyParams p) {
  uint8_t* layer = p.pool + blockIdx.z * p.layer_stride;
  const uint8_t* s = layer + p.src[blockIdx.y] * p.page_bytes;
  uint8_t* d = layer + p.dst[blockIdx.y] * p.page_bytes;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kCopyBytes + threadIdx.x * 16;
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 4096 < p.page_bytes) v[i] = __ldcs(reinterpret_cast<const uint4*>(s + at + i * 4096));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 4096 < p.page_bytes) __stcs(reinterpret_cast<uint4*>(d + at + i * 4096), v[i]);
}

// ------------------------------------------------------------------ attention of few rows
// One cluster of S CTAs per (batch row, head, 8 J query rows); the CTAs split the prefix's
// pages, the 2 warps of a CTA split a page's 64 tokens, each warp with a running maximum m,
// sum l and unnormalised output of its own, joined at the end over the warps in shared
// memory and over the CTAs through distributed shared memory, in a fixed order: no
// workspace, no second launch, no atomics.
//
// A page and head is one contiguous block: one 9216-byte bulk copy per page into a ring.
// Products run on mma m16n8k16 (bf16, f32 sums) with the keys (or V's channels) as the 16
// rows and 8 queries as the columns: the expanded cache is the A operand, which takes the
// whole of a warp's lanes even for one query, is expanded once for all J query tiles, and
// costs half the instructions of the form with queries as rows.  Among pages, the instructions
// that expand the numbers are the limit: a warp issues about 300 per 16 keys, half of them on
// the half-rate ALU pipe, and HBM rate would leave a scheduler 400 cycles for them.  With 16
// warps per SM a page and head takes 0.28 us of an SM; HBM alone would take 0.21.  16 single
// tokens over 1.3k to 10.6k keys, 32 heads: 98 us, 3.2 TB/s.  The pages are 65 us of that; the
// rest goes into uneven rows, the start of 4096 CTAs and their joins, so that over the call
// nothing is near its limit (issue 52 %, ALU 44 %, HBM 38 %; the largest stalls are barriers
// and fixed latencies).  One token over 512 keys: 6 us.  (A tcgen05 tile would need the
// expanded values written to shared memory again.)
//   S^T = K Q^T   K's values s * n are exact in bf16;
//   O^T = V^T P^T V's too.  P is rounded to bf16, the type of the product's operands, as in
//                 the dense path (0.0021 off the 64-bit result in all where the output's own
//                 rounding makes 0.0017; l sums P before the rounding, in f32); P^T comes out
//                 of S^T by two 8x8 transposes (movmatrix).
struct AttnParams4 {
  const uint8_t* pool;
  const int32_t* table;
  int32_t num_pages, max_pages;
  const __nv_bfloat16 *q, *k, *v;  // [B][H][T][128], [B][H][T][128], [B][T][H][128]
  __nv_bfloat16* out;              // [B][T][H][128]
  const b200_kv_desc* desc;
  const int32_t* row_limit;
  int32_t* status;
  int32_t heads, tokens, prefix_len, row_tiles, splits;
  float scale_log2;
};

constexpr int kMaxSplits = 8;
constexpr int kWarps = 2;                // of a CTA
constexpr int kThreads = 32 * kWarps;
constexpr int kChunks = 4 / kWarps;      // 16-key chunks of a page per warp

// J query tiles of 8 rows: a tile takes 32 registers for the output and 16 for Q.  A warp
// takes 32 keys of a page at a time: two independent chains of products hide each other's
// latency.  (4 warps of 16 keys, at as many warps per SM: 0.32 us per page and SM instead of
// 0.28 for J = 1.  J = 4 takes 0.71 against 2 * 0.38 of J = 2, and fills its rows less often.)
template <int J>
struct AttnShape {
  static constexpr int kRows = 8 * J;
  static constexpr int kRing = J == 1 ? 3 : 4;
  static constexpr int kCtas = J == 1 ? 8 : 6;                 // per SM, by registers
  static constexpr int kJoin = kWarps * kRows * kHeadDim * 4;  // the warps' outputs
  static constexpr int kUsed = kJoin + kRows * kHeadDim * 4;   // and the CTA's
  static constexpr int kSmem = kRing * kBlock > kUsed ? kRing * kBlock : kUsed;
};

// d = a b + c
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, const float (&c)[4]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]),
        "f"(c[3]));
}

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  mma_16816(d, a, b0, b1, d);
}

// 8x8 transpose of 16-bit values: lane 4g + t gives row g, columns 2t, 2t + 1 and gets row
// g of the transpose.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Shared memory of CTA `rank` of the cluster, at this CTA's address `p`.
__device__ __forceinline__ uint32_t peer_of(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}

__device__ __forceinline__ float2 peer_f32x2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ float4 peer_f32x4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

// A whole warp waits: one try, which nearly always succeeds, and the bounded wait out of line.
__device__ __noinline__ bool warp_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || warp_wait_slow(bar, parity, abort_flag);
}

// 8 channels (one uint4) as the 4 pairs (j, j + 4) of the permuted order.
__device__ __forceinline__ void pairs_of(const uint4& u, uint32_t (&pr)[4]) {
  pr[0] = prmt(u.x, u.z, 0x5410);
  pr[1] = prmt(u.x, u.z, 0x7632);
  pr[2] = prmt(u.y, u.w, 0x5410);
  pr[3] = prmt(u.y, u.w, 0x7632);
}

// A warp's softmax state.  Lane 4g + t holds queries 8j + 2t + e; o[2c + z][j][2y + e] is
// channel 32c + 4g + 2z + y of that query.  m is the same in all lanes of a t, less is -m
// (0 before the first key); l is this lane's share.
template <int J>
struct WarpState {
  float m[J][2], less[J][2], l[J][2];
  float o[8][J][4];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      m[j][0] = m[j][1] = -INFINITY;
      less[j][0] = less[j][1] = 0.f;
      l[j][0] = l[j][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int z = 0; z < 4; ++z) o[i][j][z] = 0.f;
    }
  }
};

// N times 16 keys: s[n][j][2y + e] is the product of key 8y + g of chunk n with query 8j +
// 2t + e, times `scale` (log2 units) the score; -inf where masked.  va(n, c, z, a): the V
// fragment of channels 32c + 4g + 2z + {0, 1}.  The running maximum is raised only when some
// score of the warp exceeds its query's by more than kSlack (nearly every step is spared the
// shuffles), so p <= 2^kSlack.
constexpr float kSlack = 8.f;
template <int J, int N, typename VFrag>
__device__ __forceinline__ void softmax_pv(WarpState<J>& st, float (&s)[N][J][4], float scale, VFrag va) {
  bool above = false;
  float mx[J][2];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[j][e] = fmaxf(s[0][j][e], s[0][j][2 + e]);
#pragma unroll
      for (int n = 1; n < N; ++n) mx[j][e] = fmaxf(mx[j][e], fmaxf(s[n][j][e], s[n][j][2 + e]));
      above |= mx[j][e] * scale > st.m[j][e] + kSlack;
    }
  if (__any_sync(0xffffffffu, above)) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float alpha[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float m = mx[j][e] * scale;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = fmaxf(st.m[j][e], m);
        alpha[e] = m == -INFINITY ? 1.f : ex2_approx(st.m[j][e] - m);  // no key so far
        st.m[j][e] = m;
        // before the first key: 2^(-inf - 0) = 0, not 2^(-inf + inf)
        st.less[j][e] = m == -INFINITY ? 0.f : -m;
        st.l[j][e] *= alpha[e];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int z = 0; z < 4; ++z) st.o[i][j][z] *= alpha[z & 1];
    }
  }
  uint32_t pt[N][J][2];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float p[4];
#pragma unroll
      for (int z = 0; z < 4; ++z) p[z] = ex2_approx(fmaf(s[n][j][z], scale, st.less[j][z & 1]));
      st.l[j][0] += p[0] + p[2];
      st.l[j][1] += p[1] + p[3];
      pt[n][j][0] = transpose8(bf16_pair(p[0], p[1]));
      pt[n][j][1] = transpose8(bf16_pair(p[2], p[3]));
    }
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        uint32_t a[4];
        va(n, c, z, a);
#pragma unroll
        for (int j = 0; j < J; ++j) mma_16816(st.o[2 * c + z][j], a, pt[n][j][0], pt[n][j][1]);
      }
}

__device__ __forceinline__ uint4 load16(const uint8_t* x) { return *reinterpret_cast<const uint4*>(x); }

__device__ __forceinline__ uint32_t word_of(const uint4& u, int c) {
  return c == 0 ? u.x : c == 1 ? u.y : c == 2 ? u.z : u.w;
}

// The pages of one CTA on their way into the ring: warp 0 holds the page ids, 32 at a time
// and 32 ahead, and one lane issues the copies.
struct PageFeed {
  const int32_t* ids_of;
  int ids, ids_next, h, np;

  __device__ PageFeed(const AttnParams4& p, int b, int head, int first, int pages, int lane, bool mine)
      : ids_of(p.table + static_cast<int64_t>(b) * p.max_pages + first), ids(0), ids_next(0), h(head), np(pages) {
    if (mine) {
      if (lane < np) ids = ids_of[lane];
      if (32 + lane < np) ids_next = ids_of[32 + lane];
    }
  }

  // Page j (0, 1, 2, ...) into slot j % depth; the whole of warp 0 calls it.
  __device__ __forceinline__ void issue(const AttnParams4& p, uint8_t* ring, uint64_t* full, int depth, int j,
                                        int lane) {
    if (j > 0 && (j & 31) == 0) {
      ids = ids_next;
      if (j + 32 + lane < np) ids_next = ids_of[j + 32 + lane];
    }
    const int page = __shfl_sync(0xffffffffu, ids, j & 31);
    const int slot = j % depth;
    if (page >= 0 && page < p.num_pages) {
      if (lane == 0) {
        mbar_expect_tx(full + slot, kBlock);
        bulk_load(ring + slot * kBlock, p.pool + (static_cast<int64_t>(page) * p.heads + h) * kBlock,
                  kBlock, full + slot);
      }
    } else {  // no such page: steps of 0 make its tokens read as zeros
      for (int i = lane; i < (kBlock - kKsOff) / 16; i += 32)
        *reinterpret_cast<uint4*>(ring + slot * kBlock + kKsOff + i * 16) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        report_bad_page(p.status);
        mbar_arrive(full + slot);
      }
    }
  }
};

// Q fragments of rows row0 .. row0 + nrows - 1 (zeros behind): query 8j + g, channel pairs in
// the permuted order.
template <int J>
__device__ __forceinline__ void load_q(const AttnParams4& p, int b, int h, int row0, int nrows, int g, int t,
                                       uint32_t (&qf)[8][J][2]) {
  const __nv_bfloat16* qb =
      p.q + ((static_cast<int64_t>(b) * p.heads + h) * p.tokens + row0) * kHeadDim + 8 * t;
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 x = 8 * j + g < nrows
                          ? *reinterpret_cast<const uint4*>(qb + (8 * j + g) * kHeadDim + 32 * c)
                          : make_uint4(0, 0, 0, 0);
      uint32_t pr[4];
      pairs_of(x, pr);
      qf[2 * c][j][0] = pr[0];
      qf[2 * c][j][1] = pr[1];
      qf[2 * c + 1][j][0] = pr[2];
      qf[2 * c + 1][j][1] = pr[3];
    }
}

// This call's own keys (bf16), chunks of 16: `start`, start + step, ...
template <int J>
__device__ __forceinline__ void own_keys(const AttnParams4& p, WarpState<J>& st, const uint32_t (&qf)[8][J][2],
                                         int b, int h, int row0, int nrows, int tv, int start, int step, int g,
                                         int t) {
  const int most = p.row_limit ? min(tv, max(p.row_limit[row0 + nrows - 1], 0)) : tv;
  const int chunks = (most + 15) / 16;
  const __nv_bfloat16* kb = p.k + (static_cast<int64_t>(b) * p.heads + h) * p.tokens * kHeadDim;
  const __nv_bfloat16* vb = p.v + (static_cast<int64_t>(b) * p.tokens * p.heads + h) * kHeadDim;
  const int64_t v_st = static_cast<int64_t>(p.heads) * kHeadDim;
  for (int ch = start; ch < chunks; ch += step) {
    float s[1][J][4];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int z = 0; z < 4; ++z) s[0][j][z] = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t lo[4], hi[4];
      const int k0 = ch * 16 + g, k1 = k0 + 8;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      pairs_of(k0 < tv ? *reinterpret_cast<const uint4*>(kb + static_cast<int64_t>(k0) * kHeadDim + 32 * c + 8 * t) : zero, lo);
      pairs_of(k1 < tv ? *reinterpret_cast<const uint4*>(kb + static_cast<int64_t>(k1) * kHeadDim + 32 * c + 8 * t) : zero, hi);
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const uint32_t a[4] = {lo[2 * z], hi[2 * z], lo[2 * z + 1], hi[2 * z + 1]};
#pragma unroll
        for (int j = 0; j < J; ++j) mma_16816(s[0][j], a, qf[2 * c + z][j][0], qf[2 * c + z][j][1]);
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        int lim = tv;
        if (p.row_limit) lim = min(tv, max(p.row_limit[min(row0 + 8 * j + 2 * t + e, p.tokens - 1)], 0));
        if (ch * 16 + g >= lim) s[0][j][e] = -INFINITY;
        if (ch * 16 + g + 8 >= lim) s[0][j][2 + e] = -INFINITY;
      }
    softmax_pv<J, 1>(st, s, p.scale_log2, [&](int, int c, int z, uint32_t (&a)[4]) {
      uint32_t x[4];  // keys 2t, 2t + 1 (and 8 more), channels 32c + 4g + 2z + {0, 1}
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int kk = ch * 16 + (i >> 1) * 8 + 2 * t + (i & 1);
        x[i] = kk < tv ? *reinterpret_cast<const uint32_t*>(vb + kk * v_st + 32 * c + 4 * g + 2 * z) : 0u;
      }
      a[0] = prmt(x[0], x[1], 0x5410);
      a[1] = prmt(x[0], x[1], 0x7632);
      a[2] = prmt(x[2], x[3], 0x5410);
      a[3] = prmt(x[2], x[3], 0x7632);
    });
  }
}

// The CTAs of a cluster share out the output: rank r finishes channels [128 r / S, 128 (r + 1)
// / S) of every row, adding the partial outputs up in rank order.
__device__ __forceinline__ void join_ctas(const AttnParams4& p, const float (*cta_ml)[2], const float* cta_o, int b,
                                          int h, int row0, int nrows, int rank, int S, int threads) {
  const int per = kHeadDim / S / 4;  // of 4 channels each
  for (int i = threadIdx.x; i < nrows * per; i += threads) {
    const int row = i / per, ch = rank * (kHeadDim / S) + (i % per) * 4;
    float2 ml[kMaxSplits];
    float4 x[kMaxSplits];
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r) {
      const int from = r < S ? r : rank;  // past the last CTA: anything, with weight 0
      ml[r] = peer_f32x2(peer_of(&cta_ml[row][0], from));
      x[r] = peer_f32x4(peer_of(cta_o + row * kHeadDim + ch, from));
    }
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r)
      if (r < S) m = fmaxf(m, ml[r].x);
#pragma unroll
    for (int r = 0; r < kMaxSplits; ++r)
      if (r < S) {
        // m = -inf: no key, weight 0 — or scores that were all NaN, whose NaN in l has to stay
        const float f = ml[r].x == -INFINITY ? 0.f : ex2_approx(ml[r].x - m);
        l += ml[r].x == -INFINITY ? ml[r].y : f * ml[r].y;
        acc.x = fmaf(f, x[r].x, acc.x);
        acc.y = fmaf(f, x[r].y, acc.y);
        acc.z = fmaf(f, x[r].z, acc.z);
        acc.w = fmaf(f, x[r].w, acc.w);
      }
    const float inv = 1.f / l;
    *reinterpret_cast<uint2*>(
        p.out + ((static_cast<int64_t>(b) * p.tokens + row0 + row) * p.heads + h) * kHeadDim + ch) =
        make_uint2(bf16_pair(acc.x * inv, acc.y * inv), bf16_pair(acc.z * inv, acc.w * inv));
  }
}

template <int J>
__global__ void __launch_bounds__(kThreads, AttnShape<J>::kCtas) kv4_attn_kernel(const AttnParams4 p) {
  using Shape = AttnShape<J>;
  constexpr int kRing = Shape::kRing, kRows = Shape::kRows;
  extern __shared__ __align__(128) uint8_t ring[];
  // after the last page: the warps' outputs [kWarps][kRows][128] and the CTA's [kRows][128]
  float* cta_o = reinterpret_cast<float*>(ring + Shape::kJoin);
  __shared__ float warp_ml[2][kWarps][kRows];
  __shared__ __align__(8) float cta_ml[kRows][2];
  __shared__ __align__(8) uint64_t full[kRing], empty[kRing];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int S = p.splits;
  const int rank = S > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int item = blockIdx.x / S;
  const int mt = item % p.row_tiles;
  const int h = (item / p.row_tiles) % p.heads;
  const int b = item / (p.row_tiles * p.heads);
  const int row0 = mt * kRows;
  const int nrows = min(kRows, p.tokens - row0);

  const int pv = p.desc ? min(max(p.desc[b].prefix_valid, 0), p.prefix_len) : p.prefix_len;
  const int tv = p.desc ? min(max(p.desc[b].target_valid, 0), p.tokens) : p.tokens;
  const int pages = (pv + kPage - 1) / kPage;
  const int first = static_cast<int>(static_cast<int64_t>(pages) * rank / S);
  const int np = static_cast<int>(static_cast<int64_t>(pages) * (rank + 1) / S) - first;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, kWarps);
    }
    abort_word = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  __syncthreads();

  PageFeed feed(p, b, h, first, np, lane, warp == 0);
  int issued = 0;
  if (warp == 0)
    for (; issued < np && issued < kRing; ++issued) feed.issue(p, ring, full, kRing, issued, lane);

  uint32_t qf[8][J][2];
  load_q<J>(p, b, h, row0, nrows, g, t, qf);
  WarpState<J> st;
  st.clear();
  own_keys<J>(p, st, qf, b, h, row0, nrows, tv, rank + S * warp, kWarps * S, g, t);

  // ---- the prefix's pages
  const uint32_t key_sel = (g & 1) ? 0x3232 : 0x1010;  // token g's step of a pair, twice
  bool ok = true;
  int slot = 0;
  uint32_t parity = 0;
  for (int j = 0; j < np; ++j) {
    ok = warp_wait(full + slot, parity, abort_flag);
    if (!ok) break;
    const int left = pv - (first + j) * kPage - warp * (16 * kChunks);  // valid keys from here on
    if (left > 0) {
      // chunk n of this warp: octets 2n and 2n + 1 from `at` on
      const uint8_t* at = ring + slot * kBlock + warp * (kChunks * 2 * kOctetBytes) + lane * 16;
      const uint8_t* steps = ring + slot * kBlock + kKsOff + warp * (kChunks * 2 * kOctetStepBytes);
      float s[kChunks][J][4];
#pragma unroll
      for (int n = 0; n < kChunks; ++n) {
        uint4 kw[2], ks[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          kw[y] = load16(at + (2 * n + y) * kOctetBytes);
          ks[y] = load16(steps + (2 * n + y) * kOctetStepBytes + (g >> 1) * 16);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t w0 = word_of(kw[0], c), w1 = word_of(kw[1], c), p0 = word_of(ks[0], c), p1 = word_of(ks[1], c);
          const uint32_t s0 = prmt(p0, p0, key_sel), s1 = prmt(p1, p1, key_sel);
          const uint32_t l0 = less_of(s0), l1 = less_of(s1);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const uint32_t a[4] = {expand_pair(w0, 2 * z, s0, l0), expand_pair(w1, 2 * z, s1, l1),
                                   expand_pair(w0, 2 * z + 1, s0, l0), expand_pair(w1, 2 * z + 1, s1, l1)};
#pragma unroll
            for (int i = 0; i < J; ++i) {
              const float zero[4] = {0.f, 0.f, 0.f, 0.f};
              if (c == 0 && z == 0) mma_16816(s[n][i], a, qf[0][i][0], qf[0][i][1], zero);
              else mma_16816(s[n][i], a, qf[2 * c + z][i][0], qf[2 * c + z][i][1]);
            }
          }
        }
      }
      const bool whole = left >= 16 * kChunks;
      if (!whole) {  // no score behind the last token
#pragma unroll
        for (int n = 0; n < kChunks; ++n)
#pragma unroll
          for (int i = 0; i < J; ++i)
#pragma unroll
            for (int z = 0; z < 4; ++z)
              if (16 * n + 8 * (z >> 1) + g >= left) s[n][i][z] = -INFINITY;
      }
      uint4 vw[2], vs[2];
      softmax_pv<J, kChunks>(st, s, p.scale_log2, [&](int n, int c, int z, uint32_t (&a)[4]) {
        if (c == 0 && z == 0) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            vw[y] = load16(at + kVOff + (2 * n + y) * kOctetBytes);
            vs[y] = load16(steps + (kVsOff - kKsOff) + (2 * n + y) * kOctetStepBytes + t * 16);
            if (!whole) {  // nor a V step that could be NaN
              const int key = 16 * n + 8 * y + 2 * t;
              const uint32_t keep = (key < left ? 0x0000ffffu : 0u) | (key + 1 < left ? 0xffff0000u : 0u);
              vs[y].x &= keep;
              vs[y].y &= keep;
              vs[y].z &= keep;
              vs[y].w &= keep;
            }
          }
        }
        const uint32_t v0 = word_of(vw[0], c), v1 = word_of(vw[1], c);
        const uint32_t s0 = word_of(vs[0], c), s1 = word_of(vs[1], c);
        const uint32_t l0 = less_of(s0), l1 = less_of(s1);
        a[0] = expand_pair(v0, 2 * z, s0, l0);
        a[1] = expand_pair(v0, 2 * z + 1, s0, l0);
        a[2] = expand_pair(v1, 2 * z, s1, l1);
        a[3] = expand_pair(v1, 2 * z + 1, s1, l1);
      });
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + slot);
    // refill the slot that the page before left, which every warp is done with or about to be
    if (warp == 0 && j > 0 && issued < np) {
      const int prev = slot == 0 ? kRing - 1 : slot - 1;
      ok = warp_wait(empty + prev, slot == 0 ? parity ^ 1 : parity, abort_flag);
      if (!ok) break;
      feed.issue(p, ring, full, kRing, issued, lane);
      ++issued;
    }
    if (++slot == kRing) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (!ok) {
    if (lane == 0) {
      *abort_flag = 1;
      if (p.status) atomicCAS(p.status, 0, 1);
    }
    if (warp == 0)  // copies in flight land before the ring is reused
      for (int j = max(issued - kRing, 0); j < issued; ++j) mbar_wait(full + j % kRing, (j / kRing) & 1);
  }
  __syncthreads();

  // ---- join the warps
  {
    float* wo = reinterpret_cast<float*>(ring) + warp * kRows * kHeadDim;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int q = 8 * j + 2 * t + e;
        float l = st.l[j][e];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (g == 0) {
          warp_ml[0][warp][q] = st.m[j][e];
          warp_ml[1][warp][q] = l;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<float4*>(wo + q * kHeadDim + 32 * c + 4 * g) =
              make_float4(st.o[2 * c][j][e], st.o[2 * c][j][2 + e], st.o[2 * c + 1][j][e], st.o[2 * c + 1][j][2 + e]);
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nrows * (kHeadDim / 4); i += kThreads) {
    const int row = i / (kHeadDim / 4), ch = (i % (kHeadDim / 4)) * 4;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, warp_ml[0][w][row]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      // m = -inf: no key, weight 0 — or scores that were all NaN, whose NaN in l has to stay
      const float mw = warp_ml[0][w][row];
      const float f = mw == -INFINITY ? 0.f : ex2_approx(mw - m);
      l += mw == -INFINITY ? warp_ml[1][w][row] : f * warp_ml[1][w][row];
      const float4 x = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(ring) + (w * kRows + row) * kHeadDim + ch);
      acc.x = fmaf(f, x.x, acc.x);
      acc.y = fmaf(f, x.y, acc.y);
      acc.z = fmaf(f, x.z, acc.z);
      acc.w = fmaf(f, x.w, acc.w);
    }
    if (S == 1) {
      const float inv = 1.f / l;  // no key: 0 * (1 / 0) = NaN
      __nv_bfloat16* dst =
          p.out + ((static_cast<int64_t>(b) * p.tokens + row0 + row) * p.heads + h) * kHeadDim + ch;
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(bf16_pair(acc.x * inv, acc.y * inv), bf16_pair(acc.z * inv, acc.w * inv));
    } else {
      *reinterpret_cast<float4*>(cta_o + row * kHeadDim + ch) = acc;
      if (ch == 0) {
        cta_ml[row][0] = m;
        cta_ml[row][1] = l;
      }
    }
  }
  if (S == 1) return;
  // ---- join the CTAs
  cluster_barrier();
  join_ctas(p, cta_ml, cta_o, b, h, row0, nrows, rank, S, kThreads);
  cluster_barrier();  // no CTA leaves while another reads its shared memory
}

// ------------------------------------------------------------------ attention of more rows
// 64 query rows per CTA: the kernel above repeats the expansion for every 16 rows.  Here each
// of 4 warps expands a quarter of the page into shared memory, once, in the order of the
// matrix fragments (a lane writes and reads 16 bytes, a warp 512 in a row), and then takes
// its own 16 rows over the whole page.  No join of warps; clusters split the pages as above.
// Bound by the latency of a page's two phases, with 3 CTAs per SM to fill the gaps: 1.27 us
// of an SM per page and head for 64 rows, 1.0 us for 17, against 0.38 us for each 16 rows
// above.  (Two buffers and one barrier per page at 2 CTAs per SM: 1.5 us; all 64 keys of a
// page in one softmax step: 1.30 us.)
constexpr int kTileRows = 64;
constexpr int kTileWarps = 4;
constexpr int kTileThreads = 32 * kTileWarps;
constexpr int kTileRing = 3;
constexpr int kTileCtas = 3;                       // per SM, by registers
constexpr int kFragBytes = 512;                    // one fragment of a warp
constexpr int kWideBytes = 4 * 8 * kFragBytes;     // a page's K or V: 4 chunks of 8 fragments
constexpr int kTileSmem = kTileRing * kBlock + 2 * kWideBytes;
static_assert(2 * kWideBytes >= kTileRows * kHeadDim * 4, "the CTA's outputs take the fragments' place");

__global__ void __launch_bounds__(kTileThreads, kTileCtas) kv4_attn_tile_kernel(const AttnParams4 p) {
  constexpr int J = 2;
  extern __shared__ __align__(128) uint8_t ring[];
  uint8_t* wide_k = ring + kTileRing * kBlock;
  uint8_t* wide_v = wide_k + kWideBytes;
  float* cta_o = reinterpret_cast<float*>(wide_k);  // after the last page: [kTileRows][128]
  __shared__ __align__(8) float cta_ml[kTileRows][2];
  __shared__ __align__(8) uint64_t full[kTileRing];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int S = p.splits;
  const int rank = S > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int item = blockIdx.x / S;
  const int mt = item % p.row_tiles;
  const int h = (item / p.row_tiles) % p.heads;
  const int b = item / (p.row_tiles * p.heads);
  const int cta_row0 = mt * kTileRows, cta_rows = min(kTileRows, p.tokens - cta_row0);
  const int row0 = cta_row0 + warp * 8 * J;                   // this warp's rows
  const int nrows = min(8 * J, p.tokens - row0);              // <= 0: none, it only expands

  const int pv = p.desc ? min(max(p.desc[b].prefix_valid, 0), p.prefix_len) : p.prefix_len;
  const int tv = p.desc ? min(max(p.desc[b].target_valid, 0), p.tokens) : p.tokens;
  const int pages = (pv + kPage - 1) / kPage;
  const int first = static_cast<int>(static_cast<int64_t>(pages) * rank / S);
  const int np = static_cast<int>(static_cast<int64_t>(pages) * (rank + 1) / S) - first;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kTileRing; ++i) mbar_init(full + i, 1);
    abort_word = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  __syncthreads();
  PageFeed feed(p, b, h, first, np, lane, warp == 0);
  int issued = 0;
  if (warp == 0)
    for (; issued < np && issued < kTileRing; ++issued) feed.issue(p, ring, full, kTileRing, issued, lane);

  uint32_t qf[8][J][2];
  load_q<J>(p, b, h, row0, nrows, g, t, qf);
  WarpState<J> st;
  st.clear();
  if (nrows > 0) own_keys<J>(p, st, qf, b, h, row0, nrows, tv, rank, S, g, t);

  const uint32_t key_sel = (g & 1) ? 0x3232 : 0x1010;  // token g's step of a pair, twice
  bool ok = true;
  int slot = 0;
  uint32_t parity = 0;
  for (int j = 0; j < np; ++j) {
    ok = warp_wait(full + slot, parity, abort_flag);
    // every warp is done with the page before
    ok = __syncthreads_and(ok);
    if (!ok) break;
    const int left = pv - (first + j) * kPage;  // valid keys of this page (and behind it)
    {  // expand chunk `warp`
      const uint8_t* at = ring + slot * kBlock + warp * (2 * kOctetBytes) + lane * 16;
      const uint8_t* steps = ring + slot * kBlock + kKsOff + warp * (2 * kOctetStepBytes);
      uint4 kw[2], ks[2], vw[2], vs[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        kw[y] = load16(at + y * kOctetBytes);
        ks[y] = load16(steps + y * kOctetStepBytes + (g >> 1) * 16);
        vw[y] = load16(at + kVOff + y * kOctetBytes);
        vs[y] = load16(steps + (kVsOff - kKsOff) + y * kOctetStepBytes + t * 16);
        const int key = 16 * warp + 8 * y + 2 * t;
        if (key + 1 >= left) {  // behind the last token: no V step that could be NaN
          const uint32_t keep = key < left ? 0x0000ffffu : 0u;
          vs[y].x &= keep;
          vs[y].y &= keep;
          vs[y].z &= keep;
          vs[y].w &= keep;
        }
      }
      uint8_t* to = wide_k + warp * 8 * kFragBytes + lane * 16;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t s0 = word_of(ks[0], c), s1 = word_of(ks[1], c);
        s0 = prmt(s0, s0, key_sel);
        s1 = prmt(s1, s1, key_sel);
        const uint32_t w0 = word_of(kw[0], c), w1 = word_of(kw[1], c), l0 = less_of(s0), l1 = less_of(s1);
        const uint32_t u0 = word_of(vs[0], c), u1 = word_of(vs[1], c);
        const uint32_t v0 = word_of(vw[0], c), v1 = word_of(vw[1], c), m0 = less_of(u0), m1 = less_of(u1);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          *reinterpret_cast<uint4*>(to + (2 * c + z) * kFragBytes) =
              make_uint4(expand_pair(w0, 2 * z, s0, l0), expand_pair(w1, 2 * z, s1, l1),
                         expand_pair(w0, 2 * z + 1, s0, l0), expand_pair(w1, 2 * z + 1, s1, l1));
          *reinterpret_cast<uint4*>(to + kWideBytes + (2 * c + z) * kFragBytes) =
              make_uint4(expand_pair(v0, 2 * z, u0, m0), expand_pair(v0, 2 * z + 1, u0, m0),
                         expand_pair(v1, 2 * z, u1, m1), expand_pair(v1, 2 * z + 1, u1, m1));
        }
      }
    }
    __syncthreads();  // the page is expanded, and its slot is free
    if (warp == 0 && issued < np) {
      feed.issue(p, ring, full, kTileRing, issued, lane);
      ++issued;
    }
    if (nrows > 0) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // 32 keys at a time
        if (32 * half >= left) break;
        const uint8_t* fk = wide_k + half * 16 * kFragBytes + lane * 16;
        const uint8_t* fv = wide_v + half * 16 * kFragBytes + lane * 16;
        float s[2][J][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int f = 0; f < 8; ++f) {
            const uint4 x = load16(fk + (n * 8 + f) * kFragBytes);
            const uint32_t a[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < J; ++i) {
              const float zero[4] = {0.f, 0.f, 0.f, 0.f};
              if (f == 0) mma_16816(s[n][i], a, qf[0][i][0], qf[0][i][1], zero);
              else mma_16816(s[n][i], a, qf[f][i][0], qf[f][i][1]);
            }
          }
        if (left < 32 * half + 32) {  // no score behind the last token
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < J; ++i)
#pragma unroll
              for (int z = 0; z < 4; ++z)
                if (32 * half + 16 * n + 8 * (z >> 1) + g >= left) s[n][i][z] = -INFINITY;
        }
        softmax_pv<J, 2>(st, s, p.scale_log2, [&](int n, int c, int z, uint32_t (&a)[4]) {
          const uint4 x = load16(fv + (n * 8 + 2 * c + z) * kFragBytes);
          a[0] = x.x;
          a[1] = x.y;
          a[2] = x.z;
          a[3] = x.w;
        });
      }
    }
    if (++slot == kTileRing) {
      slot = 0;
      parity ^= 1;
    }
  }
  if (!ok) {
    if (lane == 0) {
      *abort_flag = 1;
      if (p.status) atomicCAS(p.status, 0, 1);
    }
    if (warp == 0)  // copies in flight land before the CTA leaves
      for (int j = max(issued - kTileRing, 0); j < issued; ++j)
        mbar_wait(full + j % kTileRing, (j / kTileRing) & 1);
  }
  __syncthreads();  // the fragments are read; their place takes the outputs

#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int q = 8 * j + 2 * t + e;
      float l = st.l[j][e];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (q >= nrows) continue;
      const float f = S == 1 ? 1.f / l : 1.f;  // no key: 0 * (1 / 0) = NaN
      if (S > 1 && g == 0) {
        cta_ml[warp * 8 * J + q][0] = st.m[j][e];
        cta_ml[warp * 8 * J + q][1] = l;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 x = make_float4(st.o[2 * c][j][e] * f, st.o[2 * c][j][2 + e] * f, st.o[2 * c + 1][j][e] * f,
                                     st.o[2 * c + 1][j][2 + e] * f);
        if (S == 1)
          *reinterpret_cast<uint2*>(p.out + ((static_cast<int64_t>(b) * p.tokens + row0 + q) * p.heads + h) * kHeadDim +
                                    32 * c + 4 * g) = make_uint2(bf16_pair(x.x, x.y), bf16_pair(x.z, x.w));
        else
          *reinterpret_cast<float4*>(cta_o + (warp * 8 * J + q) * kHeadDim + 32 * c + 4 * g) = x;
      }
    }
  if (S == 1) return;
  cluster_barrier();
  join_ctas(p, cta_ml, cta_o, b, h, cta_row0, cta_rows, rank, S, kTileThreads);
  cluster_barrier();  // no CTA leaves while another reads its shared memory
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_view(const b200_kv4_view* c) {
  if (!c || c->num_pages < 0 || c->max_pages < 0) return B200_ERR_INVALID;
  if (c->max_pages > 0 && (!c->page_table || (reinterpret_cast<uintptr_t>(c->page_table) & 3u)))
    return B200_ERR_INVALID;
  if (c->num_pages > 0 && (!c->pool || !al16(c->pool))) return B200_ERR_INVALID;
  return B200_OK;
}

constexpr int kMaxGridYZ = 65535;
constexpr int kMaxLen = 0x7fff0000;  // positions, rounded up to pages, stay in 32 bits

// Launches kv4_load_kernel; arguments are validated.
int launch_load(const b200_kv4_view& c, const int32_t* lengths, int length_stride, void* k, void* v,
                int batch, int heads, int max_len, int32_t* status, cudaStream_t stream,
                int32_t* zero = nullptr, int n_zero = 0) {
  LoadParams p{static_cast<const uint8_t*>(c.pool), c.page_table, c.num_pages, c.max_pages, lengths,
               length_stride, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), heads,
               max_len, status, zero, n_zero};
  const dim3 grid((max_len + kPage - 1) / kPage, heads, batch);
  kv4_load_kernel<<<grid, 128, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

int sm_count() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
    return 148;
  return sms;
}

// CTAs that share one row tile's pages: as many as run at once with a page each, and no more
// than kPagesPerCta pages for one, so that rows of very different lengths even out (16 rows
// of 1.3k to 10.6k tokens, 32 heads: 215 us unsplit, 97 us by 4 and by 8); at most 8, a
// portable cluster.
constexpr int kPagesPerCta = 24;
int pick_splits(int64_t items, int prefix_len, int resident) {
  const int pages = (prefix_len + kPage - 1) / kPage;
  int s = 1;
  while (s < kMaxSplits &&
         ((2 * items * s <= static_cast<int64_t>(resident) * sm_count() && pages >= 2 * s) ||
          pages > kPagesPerCta * s))
    s *= 2;
  return s;
}

template <typename Kernel>
int launch_rows(Kernel kernel, AttnParams4 p, int rows, int resident, int threads, int smem, int batch,
                cudaStream_t stream) {
  p.row_tiles = (p.tokens + rows - 1) / rows;
  const int64_t items = static_cast<int64_t>(batch) * p.heads * p.row_tiles;
  p.splits = pick_splits(items, p.prefix_len, resident);
  if (items * p.splits > 0x7fffffff) return B200_ERR_INVALID;
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return B200_ERR_CUDA;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * p.splits));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

template <int J>
int launch_few_rows_of(const AttnParams4& p, int batch, cudaStream_t stream) {
  using Shape = AttnShape<J>;
  return launch_rows(kv4_attn_kernel<J>, p, Shape::kRows, Shape::kCtas, kThreads, Shape::kSmem, batch, stream);
}

int launch_few_rows(const b200_kv4_view& c, const void* q, const void* k, const void* v, int batch,
                    int heads, int tokens, int prefix_len, const b200_kv_desc* desc,
                    const int32_t* row_limit, float scale, void* out, int32_t* status,
                    cudaStream_t stream) {
  AttnParams4 p{};
  p.pool = static_cast<const uint8_t*>(c.pool);
  p.table = c.page_table;
  p.num_pages = c.num_pages;
  p.max_pages = c.max_pages;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.desc = desc;
  p.row_limit = row_limit;
  p.status = status;
  p.heads = heads;
  p.tokens = tokens;
  p.prefix_len = prefix_len;
  p.scale_log2 = scale * 1.4426950408889634f;
  if (tokens <= 8) return launch_few_rows_of<1>(p, batch, stream);
  // 32 heads, 33 rows against 32: 16 sequences over 512 tokens, 46 us here and 50 us there;
  // 64 rows: 54 and 65 us, over 10.6k tokens 732 and 992 us, one sequence 55 and 81 us
  if (tokens <= 32) return launch_few_rows_of<2>(p, batch, stream);
  return launch_rows(kv4_attn_tile_kernel, p, kTileRows, kTileCtas, kTileThreads, kTileSmem, batch, stream);
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

// Whether the pages are read by the kernels above or expanded for the tensor-core kernel,
// whose 256-row tiles cost the same for 1 row, behind 0.66 KB per token and head at HBM rate.
// Pages and dense, in us: 64 rows, 16 x 32 heads over 10.6k tokens 732 and 1186, 4 x 32 over
// 5k 105 and 150, over 500 22 and 23; 128 rows 1432 and 1189, 202 and 150, 35 and 23.  With
// few heads in all the dense tiles leave SMs idle: 32 heads, 128 rows, 121 and 192 over
// 10.6k, 16.2 and 18.1 over 512 — but 17 and 13 over 64, where the own keys weigh more.
bool few_rows(int64_t batch, int64_t heads, int target_len, int prefix_len) {
  return target_len <= 64 || (target_len <= 128 && batch * heads <= 64 && prefix_len / 4 >= target_len);
}

size_t dense_bytes(int batch, int heads, int prefix_len) {
  return round256(static_cast<size_t>(batch) * heads * prefix_len * kHeadDim * 2);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_kv4_store(const b200_kv4_view* c, const void* k, int64_t k_sb, int64_t k_sh,
                              int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh,
                              int64_t v_st, int32_t batch, int32_t heads, int32_t tokens,
                              int32_t head_dim, const int32_t* start, const int32_t* count,
                              int32_t* status, b200_stream_t stream) {
  if (head_dim != kHeadDim) return B200_ERR_UNSUPPORTED;
  if (batch < 0 || heads < 0 || tokens < 0) return B200_ERR_INVALID;
  int rc = check_view(c);
  if (rc != B200_OK) return rc;
  if (batch == 0 || heads == 0 || tokens == 0) return B200_OK;
  if (batch > kMaxGridYZ || heads > kMaxGridYZ) return B200_ERR_INVALID;
  if (!k || !v || !al16(k) || !al16(v)) return B200_ERR_INVALID;
  const int64_t strides[] = {k_sb, k_sh, k_st, v_sb, v_sh, v_st};
  for (int64_t s : strides)
    if (s % 8 != 0) return B200_ERR_INVALID;
  StoreParams p{static_cast<uint8_t*>(c->pool), c->page_table, c->num_pages, c->max_pages,
                static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v),
                k_sb, k_sh, k_st, v_sb, v_sh, v_st, heads, tokens, start, count, status};
  // `tokens` positions from any start touch at most this many pages
  const int64_t pages = (static_cast<int64_t>(tokens) + kPage - 2) / kPage + 1;
  kv4_store_kernel<<<dim3(static_cast<unsigned>(start ? pages : (static_cast<int64_t>(tokens) + kPage - 1) / kPage),
                          heads, batch), 128, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

extern "C" int b200_kv4_load(const b200_kv4_view* c, const int32_t* lengths, int32_t length_stride,
                             void* k_out, void* v_out, int32_t batch, int32_t heads,
                             int32_t max_len, int32_t head_dim, int32_t* status,
                             b200_stream_t stream) {
  if (head_dim != kHeadDim) return B200_ERR_UNSUPPORTED;
  if (batch < 0 || heads < 0 || max_len < 0 || length_stride < 0) return B200_ERR_INVALID;
  int rc = check_view(c);
  if (rc != B200_OK) return rc;
  if (batch == 0 || heads == 0 || max_len == 0) return B200_OK;
  if (batch > kMaxGridYZ || heads > kMaxGridYZ) return B200_ERR_INVALID;
  if (max_len > kMaxLen || max_len > static_cast<int64_t>(c->max_pages) * kPage) return B200_ERR_INVALID;
  if (!k_out || !v_out || !al16(k_out) || !al16(v_out)) return B200_ERR_INVALID;
  return launch_load(*c, lengths, length_stride, k_out, v_out, batch, heads, max_len, status,
                     static_cast<cudaStream_t>(stream));
}

extern "C" int b200_kv4_copy_pages(void* pool, int32_t layers, int64_t layer_stride,
                                   int32_t num_pages, int32_t heads, const int32_t* src,
                                   const int32_t* dst, int32_t n, b200_stream_t stream) {
  if (layers < 0 || num_pages < 0 || heads < 0 || n < 0) return B200_ERR_INVALID;
  if (layers > kMaxGridYZ || layer_stride % 16 != 0) return B200_ERR_INVALID;
  if (n == 0) return B200_OK;
  if (!src || !dst) return B200_ERR_INVALID;
  // written once, and not also read: the copies of a launch run in no order
  try {
    std::vector<uint8_t> use(static_cast<size_t>(num_pages), 0);
    for (int i = 0; i < n; ++i) {
      if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages) return B200_ERR_INVALID;
      use[src[i]] = 1;
    }
    for (int i = 0; i < n; ++i) {
      if (use[dst[i]]) return B200_ERR_INVALID;
      use[dst[i]] = 2;
    }
  } catch (...) {
    return B200_ERR_INVALID;
  }
  if (layers == 0 || heads == 0) return B200_OK;
  const int64_t page_bytes = static_cast<int64_t>(heads) * kBlock;
  if (!pool || !al16(pool)) return B200_ERR_INVALID;
  if (layers > 1 && layer_stride < page_bytes * num_pages) return B200_ERR_INVALID;
  CopyParams p{};
  p.pool = static_cast<uint8_t*>(pool);
  p.layer_stride = layer_stride;
  p.page_bytes = page_bytes;
  for (int i0 = 0; i0 < n; i0 += kPairs) {
    const int m = std::min(kPairs, n - i0);
    std::copy(src + i0, src + i0 + m, p.src);
    std::copy(dst + i0, dst + i0 + m, p.dst);
    const dim3 grid(static_cast<unsigned>((page_bytes + kCopyBytes - 1) / kCopyBytes), m, layers);
    kv4_copy_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    if (cudaGetLastError() != cudaSuccess) return B200_ERR_CUDA;
  }
  return B200_OK;
}

extern "C" int b200_kv4_attention_workspace_bytes(int32_t batch, int32_t heads, int32_t target_len,
                                                  int32_t prefix_len, size_t* bytes) {
  if (!bytes || batch < 0 || heads < 0 || target_len < 0 || prefix_len < 0) return B200_ERR_INVALID;
  *bytes = few_rows(batch, heads, target_len, prefix_len)
               ? 0
               : 2 * dense_bytes(batch, heads, prefix_len) + B200_ATTN_SPLIT_WORKSPACE_BYTES;
  return B200_OK;
}

extern "C" int b200_kv4_joint_attention(const b200_kv4_view* c, const void* q_rot, const void* k_rot,
                                        const void* v, int32_t batch, int32_t heads,
                                        int32_t target_len, int32_t prefix_len, int32_t head_dim,
                                        const b200_kv_desc* desc, const int32_t* row_limit,
                                        float scale, void* out, void* workspace,
                                        size_t workspace_bytes, int32_t* status,
                                        b200_stream_t stream_) {
  if (head_dim != kHeadDim) return B200_ERR_UNSUPPORTED;
  if (batch <= 0 || heads <= 0 || target_len < 0 || prefix_len < 0) return B200_ERR_INVALID;
  int rc = check_view(c);
  if (rc != B200_OK) return rc;
  if (prefix_len > kMaxLen || prefix_len > static_cast<int64_t>(c->max_pages) * kPage) return B200_ERR_INVALID;
  if (target_len == 0) return B200_OK;
  if (batch > kMaxGridYZ || heads > kMaxGridYZ) return B200_ERR_INVALID;
  if (!q_rot || !k_rot || !v || !out) return B200_ERR_INVALID;
  const void* ptrs[] = {q_rot, k_rot, v, out, workspace};
  for (const void* ptr : ptrs)
    if (!al16(ptr)) return B200_ERR_INVALID;
  if (!(scale > 0.f) || !std::isfinite(scale)) return B200_ERR_INVALID;
  auto stream = static_cast<cudaStream_t>(stream_);
  if (few_rows(batch, heads, target_len, prefix_len))
    return launch_few_rows(*c, q_rot, k_rot, v, batch, heads, target_len, prefix_len, desc, row_limit,
                           scale, out, status, stream);
  size_t need = 0;
  b200_kv4_attention_workspace_bytes(batch, heads, target_len, prefix_len, &need);
  if (need > 0 && (!workspace || workspace_bytes < need)) return B200_ERR_WORKSPACE;
  auto* ws = static_cast<uint8_t*>(workspace);
  const size_t one = dense_bytes(batch, heads, prefix_len);
  int n_zero = 0;
  int32_t* counters = split_counters(ws + 2 * one, &n_zero);
  if (prefix_len > 0) {
    rc = launch_load(*c, desc ? &desc[0].prefix_valid : nullptr, 2, ws, ws + one, batch, heads,
                     prefix_len, status, stream, counters, n_zero);
    if (rc != B200_OK) return rc;
  }
  return joint_attention(q_rot, k_rot, v, ws, ws + one, batch, heads, target_len, prefix_len, desc,
                         scale, out, status, ws + 2 * one, stream, prefix_len > 0, row_limit);
}

extern "C" int b200_kv4_attn_workspace_bytes(const b200_attn_args* a, size_t* bytes) {
  if (!a || !bytes) return B200_ERR_INVALID;
  if (a->batch < 0 || a->heads < 0 || a->target_len < 0 || a->prefix_len < 0) return B200_ERR_INVALID;
  size_t need = 0;
  b200_kv4_attention_workspace_bytes(a->batch, a->heads, a->target_len, a->prefix_len, &need);
  const size_t tensor =
      round256(static_cast<size_t>(a->batch) * a->heads * a->target_len * kHeadDim * 2);
  *bytes = need + tensor * (a->k_rot_out ? 1 : 2);  // post-RoPE Q, and K unless it is an output
  return B200_OK;
}

extern "C" int b200_kv4_attn_fwd(const b200_attn_args* a, const b200_kv4_view* cache,
                                 b200_stream_t stream) {
  if (!a) return B200_ERR_INVALID;
  if (a->head_dim != kHeadDim) return B200_ERR_UNSUPPORTED;
  if (a->batch <= 0 || a->heads <= 0 || a->target_len < 0 || a->prefix_len < 0) return B200_ERR_INVALID;
  int rc = check_view(cache);
  if (rc != B200_OK) return rc;
  if (a->prefix_k || a->prefix_v) return B200_ERR_INVALID;
  if (a->prefix_len > static_cast<int64_t>(cache->max_pages) * kPage) return B200_ERR_INVALID;
  if (a->target_len == 0) return B200_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->norm_q_w || !a->norm_k_w || !a->pe)
    return B200_ERR_INVALID;
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return B200_ERR_INVALID;
  if (a->pe_batch_stride < 0 || a->pe_batch_stride % 4 != 0) return B200_ERR_INVALID;
  const void* ptrs[] = {a->q, a->k, a->v, a->out, a->norm_q_w, a->norm_k_w,
                        a->pe, a->workspace, a->k_rot_out, a->v_out};
  for (const void* ptr : ptrs)
    if (!al16(ptr)) return B200_ERR_INVALID;
  size_t need = 0, inner = 0;
  b200_kv4_attn_workspace_bytes(a, &need);
  b200_kv4_attention_workspace_bytes(a->batch, a->heads, a->target_len, a->prefix_len, &inner);
  if (!a->workspace || a->workspace_bytes < need) return B200_ERR_WORKSPACE;
  const size_t tensor =
      round256(static_cast<size_t>(a->batch) * a->heads * a->target_len * kHeadDim * 2);
  auto* ws = static_cast<uint8_t*>(a->workspace);
  void* q_rot = ws + inner;
  void* k_rot = a->k_rot_out ? a->k_rot_out : ws + inner + tensor;
  rc = attn_prologue(*a, q_rot, k_rot, static_cast<cudaStream_t>(stream));
  if (rc != B200_OK) return rc;
  return b200_kv4_joint_attention(cache, q_rot, k_rot, a->v, a->batch, a->heads, a->target_len,
                                  a->prefix_len, kHeadDim, a->desc, a->row_limit, a->scale, a->out,
                                  ws, inner, a->status, stream);
}
