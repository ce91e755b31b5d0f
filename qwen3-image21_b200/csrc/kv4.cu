// kv4.cu — the paged 4-bit prefix cache of include/b200_kv4.h: store, read back, page
// copies, and attention of few query rows straight from the 4-bit pages.
//
//   kv4_store_kernel  one warp per 16 tokens of a page and head: group maxima by shuffles,
//                     numbers packed in registers, 16-byte stores in the block's order.
//   kv4_load_kernel   the inverse; s * n is exact in bf16.
//   kv4_copy_kernel   16-byte copies of page pairs passed by value.
//   kv4_attn_kernel   see there.
// All four are bound by HBM (or, at a few pages, by their launch).
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

// Nibbles i and i + 4 of w, each n + 8, as the bf16 pair (n, n): 0x4300 | u is the bf16
// number 128 + u (7 mantissa bits, one unit each), and 128 + u - 136 = n is exact.
__device__ __forceinline__ uint32_t nibble_pair(uint32_t w, int i) {
  const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
  __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&u);
  const uint32_t bias = 0x43084308u;  // (136, 136)
  v = __hsub2(v, *reinterpret_cast<const __nv_bfloat162*>(&bias));
  return *reinterpret_cast<uint32_t*>(&v);
}

// ------------------------------------------------------------------ store
// The step of a group whose largest magnitude is `top` (a bf16 value, or NaN): top / 7 cut
// to 5 significant bits.  top has 8 bits, so the rounded quotient lies on its own side of
// every 5-bit number.  Cutting, not rounding: 7 s <= top cannot overflow, and top / s < 7.44
// still has the number 7.
__device__ __forceinline__ float group_step(float top) {
  if (!(top <= 3.402823466e38f)) return __uint_as_float(0x7fc00000u);  // infinity or NaN
  if (top < kTiny) return 0.f;
  return __uint_as_float(__float_as_uint(__fdiv_rn(top, 7.f)) & 0xfff80000u);
}

// n + 8 of x for a step s > 0 (inv = 1 / s): |x| / s differs from a half by 0 or by at least
// 2^-10 (x has 8 significant bits, s has 5, n at most 3), and |x| * inv is off by less than
// 2^-20, so 2^-12 added sends exact halves up and moves no other value across one.
__device__ __forceinline__ uint32_t number(float x, float inv) {
  const int n = __float2int_rd(fmaf(fabsf(x), inv, 0.5f + 0.000244140625f));
  return static_cast<uint32_t>(x < 0.f ? 8 - n : 8 + n);
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
__global__ void __launch_bounds__(128) kv4_store_kernel(const StoreParams p) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int64_t first = p.start ? p.start[b] : 0;
  const int64_t n = p.count ? min(max(p.count[b], 0), p.tokens) : p.tokens;
  // floor division: a negative start has its tokens before page 0
  const int64_t page_i = (first >= 0 ? first / kPage : -((-first + kPage - 1) / kPage)) + blockIdx.x;
  const int64_t base = page_i * kPage + warp * 16;  // position of this warp's first token
  if (base + 16 <= first || base >= first + n) return;
  int page = -1;
  if (page_i >= 0 && page_i < p.max_pages) page = p.table[static_cast<int64_t>(b) * p.max_pages + page_i];
  if (page < 0 || page >= p.num_pages) {
    if (lane == 0) report_bad_page(p.status);
    return;
  }
  uint8_t* block = p.pool + (static_cast<int64_t>(page) * p.heads + h) * kBlock;
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
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const int octet = 2 * warp + o;
    // ---- K
    uint32_t words[4];
    float step[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t w[4] = {kx[o][c].x, kx[o][c].y, kx[o][c].z, kx[o][c].w};
      uint32_t m = mag_max(mag_max(mag_max(mag_max(0u, w[0]), w[1]), w[2]), w[3]);
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
      step[c] = group_step(__uint_as_float(max(m & 0xffffu, m >> 16) << 16));
      const bool use = step[c] > 0.f;
      const float inv = use ? __fdiv_rn(1.f, step[c]) : 0.f;
      uint32_t out = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        out |= (use ? number(bf16_lo(w[j]), inv) : 8u) << (8 * j);
        out |= (use ? number(bf16_hi(w[j]), inv) : 8u) << (8 * j + 4);
      }
      words[c] = out;
    }
    if (have(8 * o + g)) {
      *reinterpret_cast<uint4*>(block + octet * kOctetBytes + lane * 16) =
          make_uint4(words[0], words[1], words[2], words[3]);
      // lane t writes group t's step of token g = 2t' + parity
      const float s = t == 0 ? step[0] : t == 1 ? step[1] : t == 2 ? step[2] : step[3];
      reinterpret_cast<__nv_bfloat16*>(block + kKsOff + octet * kOctetStepBytes)[(g >> 1) * 8 + 2 * t + (g & 1)] =
          __float2bfloat16_rn(s);
    }
    // ---- V
    uint32_t vw[4] = {0, 0, 0, 0}, vs[4] = {0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t w[2] = {vx[o][q][c].x, vx[o][q][c].y};
        uint32_t m = mag_max(mag_max(0u, w[0]), w[1]);
        m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 16));
        const float s = group_step(__uint_as_float(max(m & 0xffffu, m >> 16) << 16));
        const bool use = s > 0.f;
        const float inv = use ? __fdiv_rn(1.f, s) : 0.f;
        uint32_t half = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          half |= (use ? number(bf16_lo(w[j]), inv) : 8u) << (8 * j);
          half |= (use ? number(bf16_hi(w[j]), inv) : 8u) << (8 * j + 4);
        }
        vw[c] |= half << (16 * q);
        vs[c] |= (__float_as_uint(s) >> 16) << (16 * q);
      }
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
};

// s * n of a nibble pair, exact in bf16.  A step that is zero keeps zeros, NaN gives NaN.
__device__ __forceinline__ uint32_t scaled(uint32_t pair, uint32_t step2) {
  const __nv_bfloat162 a = *reinterpret_cast<const __nv_bfloat162*>(&pair);
  const __nv_bfloat162 s = *reinterpret_cast<const __nv_bfloat162*>(&step2);
  const __nv_bfloat162 r = __hmul2(a, s);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// grid (page, head, batch row), lanes as in the store.
__global__ void __launch_bounds__(128) kv4_load_kernel(const LoadParams p) {
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
        const uint32_t s2 = prmt(kss[c], kss[c], (g & 1) ? 0x3232 : 0x1010);
        uint32_t pr[4];  // channels (i, i + 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = scaled(nibble_pair(kws[c], i), s2);
        const uint4 out = make_uint4(prmt(pr[0], pr[1], 0x5410), prmt(pr[2], pr[3], 0x5410),
                                     prmt(pr[0], pr[1], 0x7632), prmt(pr[2], pr[3], 0x7632));
        *reinterpret_cast<uint4*>(p.k + (row0 + rk) * kHeadDim + 32 * c + 8 * t) =
            live ? out : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // V: tokens 2t, 2t + 1, pairs (token, token + 1)
      uint32_t pr[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) pr[i] = scaled(nibble_pair(vws[c], i), vss[c]);
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
// One cluster of S CTAs per (batch row, head, 16 query rows); the CTAs split the prefix's
// pages, the 4 warps of a CTA split a page's 64 tokens, each warp with a running maximum m,
// sum l and unnormalised output of its own, joined at the end over the warps in shared
// memory and over the CTAs through distributed shared memory, in a fixed order: no
// workspace, no second launch, no atomics.
//
// Per page one 9216-byte bulk copy into a 4-deep ring (the block is contiguous); the ring
// of 3 CTAs per SM keeps about 80 KB in flight.  Products run on mma m16n8k16 (bf16, f32
// sums): at 1 to 16 rows the kernel is bound by the cache's bytes and by the instructions
// that expand them, and a tcgen05 tile would need the numbers written to shared memory
// again.  The numbers enter the products as the integers -7..7, exact in bf16:
//   score_j = scale * sum over groups c of  kstep_jc * (q_c . n_jc)
//   o_ch    = sum_j bf16(p_j * vstep_jc) * n_j,ch
// so K's expansion rounds nothing, and V's rounds p once per group as the dense path
// rounds p.  Channels are permuted alike in Q and K (and in V and the output), so that a
// lane takes its fragments with one 16-byte shared load per octet.
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

constexpr int kRows = 16;        // query rows of a CTA
constexpr int kRing = 4;
constexpr int kAttnThreads = 128;

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The shared-memory word at `addr` of CTA `rank` of the cluster.
__device__ __forceinline__ float remote_f32(const float* addr, uint32_t rank) {
  float v;
  asm volatile(
      "{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %1, %2;\n\t"
      "ld.shared::cluster.f32 %0, [ra];\n\t}"
      : "=f"(v)
      : "r"(smem_addr(addr)), "r"(rank)
      : "memory");
  return v;
}

// 8 channels (one uint4) as the 4 pairs (j, j + 4) of the permuted order.
__device__ __forceinline__ void pairs_of(const uint4& u, uint32_t (&pr)[4]) {
  pr[0] = prmt(u.x, u.z, 0x5410);
  pr[1] = prmt(u.x, u.z, 0x7632);
  pr[2] = prmt(u.y, u.w, 0x5410);
  pr[3] = prmt(u.y, u.w, 0x7632);
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// A warp's softmax state: lane 4g + t holds rows g and g + 8; o[4c + i] is the output tile
// whose column 2t + e is channel 32c + 8t + 4e + i.
struct WarpState {
  float m[2], l[2];
  float o[16][4];
};

// 16 keys: s[a][2r + e] is the score (log2 units) of row g + 8r and key 8a + 2t + e, -inf
// where masked; vstep[a][c] the V steps of keys 2t, 2t + 1 of octet a as a bf16 pair;
// vpair(a, c, i) the V fragment of octet a, group c, channel i.
template <typename VPair>
__device__ __forceinline__ void softmax_pv(WarpState& st, float (&s)[2][4], const uint32_t (&vstep)[2][4],
                                           VPair vpair) {
  float p[2][4], ref[2], alpha[2];
  bool moved = false;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float mx =
        quad_max(fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])));
    const float m = fmaxf(st.m[r], mx);
    moved |= m != st.m[r];
    ref[r] = m == -INFINITY ? 0.f : m;  // no key so far: 2^(-inf - 0) = 0, not NaN
    alpha[r] = ex2_approx(st.m[r] - ref[r]);
    st.m[r] = m;
  }
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) p[a][i] = ex2_approx(s[a][i] - ref[i >> 1]);
  if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[i][e] *= alpha[e >> 1];
    st.l[0] *= alpha[0];
    st.l[1] *= alpha[1];
  }
#pragma unroll
  for (int r = 0; r < 2; ++r)
    st.l[r] += (p[0][2 * r] + p[0][2 * r + 1]) + (p[1][2 * r] + p[1][2 * r + 1]);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t a[4];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const float v0 = bf16_lo(vstep[o][c]), v1 = bf16_hi(vstep[o][c]);
      a[2 * o] = bf16_pair(p[o][0] * v0, p[o][1] * v1);
      a[2 * o + 1] = bf16_pair(p[o][2] * v0, p[o][3] * v1);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) mma_16816(st.o[4 * c + i], a, vpair(0, c, i), vpair(1, c, i));
  }
}

__global__ void __launch_bounds__(kAttnThreads, 3) kv4_attn_kernel(const AttnParams4 p) {
  // The ring; after the last page, the warps' outputs [4][16][128].
  __shared__ __align__(128) uint8_t ring[kRing * kBlock];
  __shared__ __align__(16) float cta_o[kRows * kHeadDim];
  __shared__ float warp_ml[2][4][kRows];
  __shared__ float cta_ml[2][kRows];
  __shared__ __align__(8) uint64_t full[kRing], empty[kRing];
  __shared__ int page_ok[kRing];
  __shared__ int abort_word;
  static_assert(kRing * kBlock >= 4 * kRows * kHeadDim * 4, "the ring holds the warps' outputs");
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
      mbar_init(empty + i, 4);
    }
    abort_word = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  __syncthreads();

  // Warp 0 keeps the ring filled: page ids by 32 at a time, one lane issues.
  const int32_t* ids_of = p.table + static_cast<int64_t>(b) * p.max_pages + first;
  int ids = 0, ids_next = 0;
  if (warp == 0) {
    if (lane < np) ids = ids_of[lane];
    if (32 + lane < np) ids_next = ids_of[32 + lane];
  }
  auto issue = [&](int j) {  // warp 0, j = 0, 1, 2, ...
    if (j > 0 && (j & 31) == 0) {
      ids = ids_next;
      if (j + 32 + lane < np) ids_next = ids_of[j + 32 + lane];
    }
    const int page = __shfl_sync(0xffffffffu, ids, j & 31);
    if (lane == 0) {
      const int slot = j % kRing;
      const bool ok = page >= 0 && page < p.num_pages;
      page_ok[slot] = ok;
      if (ok) {
        mbar_expect_tx(full + slot, kBlock);
        bulk_load(ring + slot * kBlock, p.pool + (static_cast<int64_t>(page) * p.heads + h) * kBlock,
                  kBlock, full + slot);
      } else {
        report_bad_page(p.status);
        mbar_arrive(full + slot);
      }
    }
  };
  int issued = 0;
  if (warp == 0)
    for (; issued < np && issued < kRing; ++issued) issue(issued);

  // Q fragments: rows g and g + 8 (zeros behind the last row)
  uint32_t qf[8][4];
  {
    const __nv_bfloat16* qb =
        p.q + ((static_cast<int64_t>(b) * p.heads + h) * p.tokens + row0) * kHeadDim + 8 * t;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t lo[4], hi[4];
      const uint4 zero = make_uint4(0, 0, 0, 0);
      pairs_of(g < nrows ? *reinterpret_cast<const uint4*>(qb + g * kHeadDim + 32 * c) : zero, lo);
      pairs_of(g + 8 < nrows ? *reinterpret_cast<const uint4*>(qb + (g + 8) * kHeadDim + 32 * c) : zero, hi);
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        qf[2 * c + z][0] = lo[2 * z];
        qf[2 * c + z][1] = hi[2 * z];
        qf[2 * c + z][2] = lo[2 * z + 1];
        qf[2 * c + z][3] = hi[2 * z + 1];
      }
    }
  }
  WarpState st;
  st.m[0] = st.m[1] = -INFINITY;
  st.l[0] = st.l[1] = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) st.o[i][e] = 0.f;

  // ---- this call's own keys (bf16), 16 at a time, dealt out over CTAs and warps
  {
    int lim[2] = {tv, tv};
    int most = tv;
    if (p.row_limit) {
#pragma unroll
      for (int r = 0; r < 2; ++r)
        lim[r] = min(tv, max(p.row_limit[min(row0 + g + 8 * r, p.tokens - 1)], 0));
      most = min(tv, max(p.row_limit[row0 + nrows - 1], 0));
    }
    const int chunks = (most + 15) / 16;
    const __nv_bfloat16* kb = p.k + (static_cast<int64_t>(b) * p.heads + h) * p.tokens * kHeadDim;
    const __nv_bfloat16* vb = p.v + (static_cast<int64_t>(b) * p.tokens * p.heads + h) * kHeadDim;
    const int64_t v_st = static_cast<int64_t>(p.heads) * kHeadDim;
    for (int ch = rank + S * warp; ch < chunks; ch += 4 * S) {
      float s[2][4];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int key = ch * 16 + 8 * a + g;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pr[4];
          pairs_of(key < tv ? *reinterpret_cast<const uint4*>(kb + static_cast<int64_t>(key) * kHeadDim + 32 * c + 8 * t)
                            : make_uint4(0, 0, 0, 0), pr);
          mma_16816(acc, qf[2 * c], pr[0], pr[1]);
          mma_16816(acc, qf[2 * c + 1], pr[2], pr[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kk = ch * 16 + 8 * a + 2 * t + (i & 1);
          s[a][i] = kk < lim[i >> 1] ? acc[i] * p.scale_log2 : -INFINITY;
        }
      }
      const uint32_t one = 0x3f803f80u;
      const uint32_t vstep[2][4] = {{one, one, one, one}, {one, one, one, one}};
      uint2 vx[2][2][4];  // [octet][parity][group]: channels 32c + 4g + 0..3
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int kk = ch * 16 + 8 * a + 2 * t + e;
            vx[a][e][c] = kk < tv ? *reinterpret_cast<const uint2*>(vb + kk * v_st + 32 * c + 4 * g)
                                  : make_uint2(0, 0);
          }
      softmax_pv(st, s, vstep, [&](int a, int c, int i) {
        const uint2 x0 = vx[a][0][c], x1 = vx[a][1][c];
        return prmt(i < 2 ? x0.x : x0.y, i < 2 ? x1.x : x1.y, (i & 1) ? 0x7632 : 0x5410);
      });
    }
  }

  // ---- the prefix's pages
  bool ok = true;
  for (int j = 0; j < np; ++j) {
    const int slot = j % kRing;
    ok = __all_sync(0xffffffffu, mbar_wait(full + slot, (j / kRing) & 1, abort_flag));
    if (!ok) break;
    const uint8_t* blk = ring + slot * kBlock;
    const bool good = page_ok[slot] != 0;
    const int left = pv - (first + j) * kPage - warp * 16;  // valid keys from this chunk on
    if (left > 0) {
      float s[2][4];
      uint32_t vstep[2][4];
      uint4 vw[2];
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const int octet = 2 * warp + a;
        const uint4 kw4 = *reinterpret_cast<const uint4*>(blk + octet * kOctetBytes + lane * 16);
        uint4 ks4 = *reinterpret_cast<const uint4*>(blk + kKsOff + octet * kOctetStepBytes + t * 16);
        uint4 vs4 = *reinterpret_cast<const uint4*>(blk + kVsOff + octet * kOctetStepBytes + t * 16);
        vw[a] = *reinterpret_cast<const uint4*>(blk + kVOff + octet * kOctetBytes + lane * 16);
        if (!good) ks4 = vs4 = make_uint4(0, 0, 0, 0);  // reads as zeros
        const uint32_t kw[4] = {kw4.x, kw4.y, kw4.z, kw4.w};
        const uint32_t ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w};
        vstep[a][0] = vs4.x;
        vstep[a][1] = vs4.y;
        vstep[a][2] = vs4.z;
        vstep[a][3] = vs4.w;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[a][i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816(acc, qf[2 * c], nibble_pair(kw[c], 0), nibble_pair(kw[c], 1));
          mma_16816(acc, qf[2 * c + 1], nibble_pair(kw[c], 2), nibble_pair(kw[c], 3));
          const float s0 = bf16_lo(ks[c]) * p.scale_log2, s1 = bf16_hi(ks[c]) * p.scale_log2;
          s[a][0] = fmaf(acc[0], s0, s[a][0]);
          s[a][1] = fmaf(acc[1], s1, s[a][1]);
          s[a][2] = fmaf(acc[2], s0, s[a][2]);
          s[a][3] = fmaf(acc[3], s1, s[a][3]);
        }
      }
      if (left < 16) {  // behind the last token: no score, and no V step that could be NaN
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (8 * a + 2 * t + e >= left) {
              s[a][e] = s[a][2 + e] = -INFINITY;
#pragma unroll
              for (int c = 0; c < 4; ++c) vstep[a][c] &= e ? 0x0000ffffu : 0xffff0000u;
            }
      }
      softmax_pv(st, s, vstep, [&](int a, int c, int i) {
        const uint32_t w = c == 0 ? vw[a].x : c == 1 ? vw[a].y : c == 2 ? vw[a].z : vw[a].w;
        return nibble_pair(w, i);
      });
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + slot);
    // refill the slot that the page before left, which every warp is done with or about to be
    if (warp == 0 && j > 0 && issued < np) {
      ok = __all_sync(0xffffffffu, mbar_wait(empty + (j - 1) % kRing, ((j - 1) / kRing) & 1, abort_flag));
      if (!ok) break;
      issue(issued++);
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
    for (int r = 0; r < 2; ++r) {
      const float l = quad_sum(st.l[r]);
      if (t == 0) {
        warp_ml[0][warp][g + 8 * r] = st.m[r];
        warp_ml[1][warp][g + 8 * r] = l;
      }
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float4*>(wo + (g + 8 * r) * kHeadDim + 32 * c + 8 * t + 4 * e) =
              make_float4(st.o[4 * c][2 * r + e], st.o[4 * c + 1][2 * r + e], st.o[4 * c + 2][2 * r + e],
                          st.o[4 * c + 3][2 * r + e]);
    }
  }
  __syncthreads();
  const int row = threadIdx.x >> 3;
  if (row < nrows) {
    float m = -INFINITY, l = 0.f, w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, warp_ml[0][i][row]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float mi = warp_ml[0][i][row];
      w[i] = mi == -INFINITY ? 0.f : ex2_approx(mi - m);
      // a warp whose scores were all NaN keeps m = -inf and l = NaN: that NaN has to stay
      l += mi == -INFINITY ? warp_ml[1][i][row] : w[i] * warp_ml[1][i][row];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int ch = (threadIdx.x & 7) * 4 + 32 * k;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(
            reinterpret_cast<const float*>(ring) + (i * kRows + row) * kHeadDim + ch);
        acc.x = fmaf(w[i], x.x, acc.x);
        acc.y = fmaf(w[i], x.y, acc.y);
        acc.z = fmaf(w[i], x.z, acc.z);
        acc.w = fmaf(w[i], x.w, acc.w);
      }
      *reinterpret_cast<float4*>(cta_o + row * kHeadDim + ch) = acc;
    }
    if ((threadIdx.x & 7) == 0) {
      cta_ml[0][row] = m;
      cta_ml[1][row] = l;
    }
  }
  // ---- join the CTAs: rank r finishes channels [128 r / S, 128 (r + 1) / S) of every row
  if (S > 1) cluster_barrier();
  else __syncthreads();
  if (row < nrows) {
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < S; ++i) m = fmaxf(m, S > 1 ? remote_f32(&cta_ml[0][row], i) : cta_ml[0][row]);
    for (int i = 0; i < S; ++i) {
      const float mi = S > 1 ? remote_f32(&cta_ml[0][row], i) : cta_ml[0][row];
      const float li = S > 1 ? remote_f32(&cta_ml[1][row], i) : cta_ml[1][row];
      l += mi == -INFINITY ? li : ex2_approx(mi - m) * li;
    }
    const float inv = 1.f / l;  // no key: 0 * (1 / 0) = NaN
    const int per = kRows / S;  // channels of this thread
    __nv_bfloat16* dst =
        p.out + ((static_cast<int64_t>(b) * p.tokens + row0 + row) * p.heads + h) * kHeadDim;
    for (int k = 0; k < per; ++k) {
      const int ch = rank * (kHeadDim / S) + (threadIdx.x & 7) + 8 * k;
      float acc = 0.f;
      for (int i = 0; i < S; ++i) {
        const float mi = S > 1 ? remote_f32(&cta_ml[0][row], i) : cta_ml[0][row];
        const float w = mi == -INFINITY ? 0.f : ex2_approx(mi - m);
        const float x = S > 1 ? remote_f32(cta_o + row * kHeadDim + ch, i) : cta_o[row * kHeadDim + ch];
        acc = fmaf(w, x, acc);
      }
      dst[ch] = __float2bfloat16_rn(acc * inv);
    }
  }
  if (S > 1) cluster_barrier();  // no CTA leaves while another reads its shared memory
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
                int batch, int heads, int max_len, int32_t* status, cudaStream_t stream) {
  LoadParams p{static_cast<const uint8_t*>(c.pool), c.page_table, c.num_pages, c.max_pages, lengths,
               length_stride, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), heads,
               max_len, status};
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

// CTAs that share one row tile's pages: enough that the launch fills the GPU (3 CTAs per
// SM), at most 8 (a portable cluster), and no fewer than 2 pages each.
int pick_splits(int64_t items, int prefix_len) {
  const int pages = (prefix_len + kPage - 1) / kPage;
  int s = 1;
  while (s < 8 && items * s < 3 * sm_count() && pages >= 4 * s) s *= 2;
  return s;
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
  p.row_tiles = (tokens + kRows - 1) / kRows;
  p.scale_log2 = scale * 1.4426950408889634f;
  const int64_t items = static_cast<int64_t>(batch) * heads * p.row_tiles;
  p.splits = pick_splits(items, prefix_len);
  if (items * p.splits > 0x7fffffff) return B200_ERR_INVALID;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * p.splits));
  cfg.blockDim = dim3(kAttnThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_attn_kernel, p);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? B200_OK : B200_ERR_CUDA;
}

size_t round256(size_t x) { return (x + 255) / 256 * 256; }

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
  *bytes = target_len < B200_KV4_DENSE_QUERIES
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
  if (target_len < B200_KV4_DENSE_QUERIES)
    return launch_few_rows(*c, q_rot, k_rot, v, batch, heads, target_len, prefix_len, desc, row_limit,
                           scale, out, status, stream);
  size_t need = 0;
  b200_kv4_attention_workspace_bytes(batch, heads, target_len, prefix_len, &need);
  if (need > 0 && (!workspace || workspace_bytes < need)) return B200_ERR_WORKSPACE;
  auto* ws = static_cast<uint8_t*>(workspace);
  const size_t one = dense_bytes(batch, heads, prefix_len);
  if (prefix_len > 0) {
    rc = launch_load(*c, desc ? &desc[0].prefix_valid : nullptr, 2, ws, ws + one, batch, heads,
                     prefix_len, status, stream);
    if (rc != B200_OK) return rc;
  }
  return joint_attention(q_rot, k_rot, v, ws, ws + one, batch, heads, target_len, prefix_len, desc,
                         scale, out, status, ws + 2 * one, stream, false, row_limit);
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
