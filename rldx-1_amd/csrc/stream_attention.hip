// Attention over a stream of tokens: a sliding window with sinks over bf16 K/V rows
// (rldx_window_attention_bf16) and over the 4-bit paged cache (rldx_kv4_attention_bf16).
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax over the visible j of (q_i . k_j scale);
//   j is visible to a query at p iff j <= p and (j > p - window or j < sinks).
//
// rows_attn_kernel: few query rows per KV head (single tokens, chunks).  The rows of a KV head's
// whole group, (token, head) pairs in that order, are the 16 columns of S^T = K Q^T, so K and V
// are read once for the group.  Per 32 keys a wave runs
//   S^T  = K Q^T  two 16-key blocks, v_mfma_f32_16x16x32_bf16 over head_dim
//   O^T += V^T P^T  one 32-key step for each of head_dim / 16 blocks of dimensions
// and P^T goes from the S^T accumulators to the B operand without leaving its lane: lane group g
// holds keys 4 g .. 4 g + 3 of both blocks, and the V^T operand takes its 32 keys in that order.
// V rows are turned by v_perm on pairs of rows that the lane itself has loaded (8 keys by head_dim / 16
// dimensions a lane), so nothing goes through LDS but the merge of the workgroup's 4 or 8 waves, which
// walk tiles w, w + 4 (8), ...  Where the rows leave most CUs idle, `splits` workgroups share
// the tiles of a row block and merge_kernel adds up their partial states (fp32, as the softmax
// reference, the sum and the unnormalised O).
#include <algorithm>

#include "kv4_cache.h"
#include "rldx_amd.h"

namespace rldx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = kv4::kTile;
constexpr int kWaves = 4;
constexpr int kRowsBlock = 16;  // rows of a rows_attn_kernel workgroup
constexpr int kMaxSplits = 64;
constexpr int kMaxSlots = 1 << 30;
constexpr float kMoveRef = 5.f;  // log2 units: the softmax reference moves when a score exceeds it by 2^5

struct StreamArgs {
  const uint16_t* q;
  int64_t q_sb, q_ss, q_sh;
  uint16_t* o;
  int64_t o_sb, o_ss, o_sh;
  // bf16 rows
  const uint16_t *k, *v;
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  const float* mask;  // [batch, sk] or null
  int64_t mask_sb;
  // 4-bit cache
  const uint8_t* cache;
  int64_t page_stride, head_stride;  // bytes
  int num_pages, page_shift;
  const int32_t* table;
  int64_t table_sb;
  const int32_t* starts;
  const int32_t* counts;  // or null
  int limit;              // readable keys: seq_k, or the slots of a row of the table
  int batch, sq, hq, hkv, group, window, sinks;
  int row_tiles, splits;
  DivMagic d_group, d_hkv, d_row_tiles, d_splits, d_items;
  float scale_log2;
  float* part;  // [batch hkv row_tiles splits][rows per tile][D] O, then the same rows' {reference, sum}
};

// The queries i0 .. i1 of a row block that see anything, and the tiles that hold what they see.
struct Span {
  int start;   // slot of query 0
  int count;   // queries i >= count see nothing
  int p0, p1;  // slots of the first and the last query of the block that sees anything, p1 < limit
  int ns, w0;  // tiles [0, ns) hold the sinks, tiles from w0 (>= ns) on the window
  int n;       // tiles in all
};

__device__ __forceinline__ int query_of(const StreamArgs& a, int row) {
  return static_cast<int>(div_u32(static_cast<uint32_t>(row), a.d_group));
}
// id / d, and the rest of it into id
__device__ __forceinline__ int split_off(int& id, int d, const DivMagic& by) {
  const int q = static_cast<int>(div_u32(static_cast<uint32_t>(id), by));
  const int rest = id - q * d;
  id = q;
  return rest;
}

template <bool kCache>
__device__ __forceinline__ Span span_of(const StreamArgs& a, int b, int row0, int rows) {
  Span s;
  s.count = a.sq;
  if constexpr (kCache) {
    s.start = min(max(__builtin_amdgcn_readfirstlane(a.starts[b]), -kMaxSlots), kMaxSlots);
    if (a.counts) s.count = min(s.count, __builtin_amdgcn_readfirstlane(a.counts[b]));
  } else {
    s.start = a.limit - a.sq;
  }
  const int i0 = max(query_of(a, row0), -min(s.start, 0));
  const int i1 = min(query_of(a, row0 + rows - 1), s.count - 1);
  s.p0 = s.start + i0;
  s.p1 = min(s.start + i1, a.limit - 1);  // (a query past the limit is NaN whatever it sees)
  if (i1 < i0 || s.p1 < s.p0) {
    s.p0 = 0;
    s.p1 = -1;
    s.ns = s.w0 = s.n = 0;
    return s;
  }
  s.ns = (min(a.sinks, s.p1 + 1) + kTile - 1) / kTile;
  s.w0 = max(s.ns, max(0, s.p0 - a.window + 1) / kTile);
  s.n = s.ns + max(0, s.p1 / kTile + 1 - s.w0);
  return s;
}

// Splits that a row block of n tiles uses: none with less than one tile for each wave.
__device__ __forceinline__ int splits_of(int splits, int n) { return max(1, min(splits, (n + kWaves - 1) / kWaves)); }
// First tile of split x of use (n <= 2^25 tiles, x <= use <= 64)
__device__ __forceinline__ int split_start(int n, int x, int use) {
  return static_cast<int>(static_cast<uint32_t>(n) * static_cast<uint32_t>(x) / static_cast<uint32_t>(use));
}

// over the 4 lanes of a query (lanes l, l ^ 16, l ^ 32, l ^ 48): the swaps leave a lane's own value and its
// partner's in the two registers
__device__ __forceinline__ float quad_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  x = fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  x = __builtin_bit_cast(float, a0) + __builtin_bit_cast(float, a1);
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
}

// What a lane loads of a tile of 32 keys.
template <int D, bool kCache>
struct Raw;
template <int D>
struct Raw<D, true> {
  u32x4 k[2];     // D = 64: two dwords of each
  u32x4 v[2];     // D = 64: the first
  uint32_t ks[2];
  u32x2 vs;
};
template <int D>
struct Raw<D, false> {
  u32x4 k[2][D / 32];
  u32x4 v[8];  // D = 64: two dwords of each
  float m[2][4];
};

__device__ __forceinline__ bf16x8 dequant8(uint32_t c, float s) {
  const u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
  return __builtin_bit_cast(bf16x8, r);
}

// (The instructions of these are opaque to the compiler, or it works them out ahead for every tile, and keeps registers
// for them, though only a few tiles come here.)
// Whether any of the bf16 values looked at is an infinity or a NaN: 0 times it is a NaN.  Looked at as fp16 pairs, one
// instruction for two: exponents from 0xf8 on count as well, values of 2^121 and more, which the caller tells apart.
struct Finite {
  uint32_t sum = 0;
  __device__ __forceinline__ void look(uint32_t w) { asm volatile("v_pk_fma_f16 %0, %1, 0, %0" : "+v"(sum) : "v"(w)); }
  __device__ __forceinline__ bool broken() const { return (sum & 0x7fffu) > 0x7c00u || (sum & 0x7fff0000u) > 0x7c000000u; }
};
__device__ __forceinline__ uint32_t finite2(uint32_t w) {  // with zeros in the place of what is not
  asm volatile("" : "+v"(w));
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}
// The keys 0 .. 31 of a tile that a query sees, a bit each: k0 <= p, and k0 > p - window or k0 < sinks.
// s where bit c is set, else -inf
__device__ __forceinline__ float seen_or_none(float s, uint32_t bits, int c) {
  const uint32_t m = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(bits), c, 1));
  return __builtin_bit_cast(float, (m & __builtin_bit_cast(uint32_t, s)) | (~m & 0xff800000u));
}
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }
__device__ __forceinline__ uint32_t visible_bits(int k0, int p, int window, int sinks) {
  return below(p + 1 - k0) & (~below(p + 1 - window - k0) | below(sinks - k0));
}

// Factor of a state whose reference moves from m to n >= m.  Never 0: an infinity in O has to stay one, and what is
// scaled by 2^-126 is lost beside the new terms just as well.  (No reference yet: O and the sum are 0.)
__device__ __forceinline__ float rescale(float m, float n) { return __builtin_amdgcn_exp2f(fmaxf(m - n, -126.f)); }
// 1 / sum of a softmax: a query that has seen nothing has O = 0; a NaN stays.
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : l == 0.f ? 1.f : l; }

template <int D, bool kCache, int NW>
__global__ __launch_bounds__(64 * NW, 2) void rows_attn_kernel(StreamArgs a) {
  constexpr int KS = D / 32;  // MFMA steps over head_dim
  constexpr int W = D / 16;   // dimensions of a lane's V columns, blocks of O^T
  constexpr int OP = D + 4;   // pitch of O in LDS (floats)
  __shared__ __attribute__((aligned(16))) float sm_o[NW][kRowsBlock][OP];
  __shared__ float sm_ml[NW][kRowsBlock][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int n16 = lane & 15, g = lane >> 4;

  // work item: (batch, kv head, split)
  int b = static_cast<int>(blockIdx.x);
  const int split = split_off(b, a.splits, a.d_splits), hk = split_off(b, a.hkv, a.d_hkv);

  const int rows = a.sq * a.group;  // <= kRowsBlock
  const Span sp = span_of<kCache>(a, b, 0, rows);
  const int use = splits_of(a.splits, sp.n);
  if (split >= use) return;
  const int t0 = split_start(sp.n, split, use), t1 = split_start(sp.n, split + 1, use);
  const int mine = t1 - t0 > wave ? (t1 - t0 - wave + NW - 1) / NW : 0;  // tiles t0 + wave + NW it
  auto tile_at = [&](int it) {
    const int t = t0 + wave + NW * it;
    return t < sp.ns ? t : sp.w0 + (t - sp.ns);
  };

  // this lane's query: column n16 (the columns past the last row repeat it, and are not stored)
  const int row = min(n16, rows - 1);
  const int qi = query_of(a, row), qh = hk * a.group + row - qi * a.group;
  const int pos = qi < sp.count ? max(sp.start + qi, -1) : -1;  // slot, -1: sees nothing
  // every query sees something
  const bool all_rows = sp.p0 == sp.start && sp.p1 == sp.start + a.sq - 1;
  bf16x8 qf[KS];
  {
    const uint16_t* const src = a.q + b * a.q_sb + qi * a.q_ss + qh * a.q_sh + (kCache ? D / 4 : 8) * g;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(src + (kCache ? 8 : 32) * s));
  }

  // page ids of the wave's next 64 tiles, one a lane
  int ids = -1, ids_base = 0;
  auto load_ids = [&](int it0) {
    ids_base = it0;
    ids = -1;
    if constexpr (kCache) {
      const int it = it0 + lane;
      if (it < mine) ids = a.table[b * a.table_sb + ((tile_at(it) * kTile) >> a.page_shift)];
    }
  };
  load_ids(0);
  auto page_of = [&](int it) {  // called with it ascending
    if (it - ids_base >= 64) load_ids(it);
    return __builtin_amdgcn_readlane(ids, it - ids_base);
  };

  auto load = [&](Raw<D, kCache>& raw, int it, int& page) {
    const int k0 = tile_at(it) * kTile;
    if constexpr (kCache) {
      page = page_of(it);
      if (page < 0 || page >= a.num_pages) {
        page = -1;
        raw = Raw<D, true>{};
        return;
      }
      const uint8_t* const t = a.cache + page * a.page_stride + hk * a.head_stride +
                               ((k0 & ((1 << a.page_shift) - 1)) / kTile) * kv4::tile_bytes(D);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int r = kt * 16 + n16;
        if constexpr (D == 128) {
          raw.k[kt] = *reinterpret_cast<const u32x4*>(t + r * 64 + g * 16);
          raw.ks[kt] = t[32 * D + r * 4 + g];
        } else {
          const u32x2 c = *reinterpret_cast<const u32x2*>(t + r * 32 + g * 8);
          raw.k[kt] = u32x4{c[0], c[1], 0, 0};
          raw.ks[kt] = t[32 * D + r * 2 + (g >> 1)];
        }
      }
      raw.v[0] = *reinterpret_cast<const u32x4*>(t + 16 * D + lane * (D / 4));
      if constexpr (D == 128) raw.v[1] = *reinterpret_cast<const u32x4*>(t + 16 * D + lane * (D / 4) + 16);
      raw.vs = *reinterpret_cast<const u32x2*>(t + 33 * D + ((n16 * W / 32) * 4 + g) * 8);
    } else {
      page = 0;
      const int last = a.limit - 1;
      const uint16_t* const kb = a.k + b * a.k_sb + hk * a.k_sh;
      const uint16_t* const vb = a.v + b * a.v_sb + hk * a.v_sh + n16 * W;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const uint16_t* const src = kb + min(k0 + kt * 16 + n16, last) * a.k_ss + g * 8;
#pragma unroll
        for (int s = 0; s < KS; ++s) raw.k[kt][s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t* const src = vb + min(k0 + (i >> 2) * 16 + g * 4 + (i & 3), last) * a.v_ss;
        if constexpr (D == 128) {
          raw.v[i] = *reinterpret_cast<const u32x4*>(src);
        } else {
          const u32x2 x = *reinterpret_cast<const u32x2*>(src);
          raw.v[i] = u32x4{x[0], x[1], 0, 0};
        }
      }
      if (a.mask) {
        const float* const m = a.mask + b * a.mask_sb;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) raw.m[kt][r] = m[min(k0 + kt * 16 + g * 4 + r, last)];
      }
    }
  };

  floatx4 oacc[W];
#pragma unroll
  for (int j = 0; j < W; ++j) oacc[j] = floatx4{0, 0, 0, 0};
  float m_ref = -__builtin_inff(), l = 0.f;
  bool odd_v = false;
  auto whole = [&](int k0) {
    return all_rows && k0 + kTile - 1 <= sp.p0 && (k0 > sp.p1 - a.window || k0 + kTile <= a.sinks);
  };

  auto compute = [&](Raw<D, kCache>& raw, int it, int page) {
    const int k0 = tile_at(it) * kTile;
    // every query sees all 32 keys: no masks, and no key whose V may not be touched
    bool full = page >= 0 && whole(k0);
    if constexpr (!kCache) {
      if (a.mask) {
        bool any = false, all = true;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            any |= raw.m[kt][r] != 0.f;
            all &= raw.m[kt][r] != 0.f;
          }
        if (!__any(any)) return;
        full = full && __all(all);
      }
    }
    // ---- S^T ----
    floatx4 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = floatx4{0, 0, 0, 0};
      float ks = 0.f;
      if constexpr (kCache) ks = __builtin_bit_cast(float, raw.ks[kt] << 23);
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        bf16x8 kf;
        if constexpr (kCache) {
          const uint32_t c = raw.k[kt][st];
          kf = dequant8(c, ks);
        } else {
          kf = __builtin_bit_cast(bf16x8, raw.k[kt][st]);
        }
        s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[st], s[kt], 0, 0, 0);
      }
    }
    // ---- visibility ----
    bool zero = false;  // (wave-uniform) V holds infinities or NaN that not every query sees
    if (!full) {
      uint32_t mbits = ~0u;  // bits 4 g .. + 3 and 16 + 4 g .. + 3: the others are not looked at
      if constexpr (!kCache) {
        if (a.mask) {
          mbits = 0;
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) mbits |= (raw.m[kt][r] != 0.f ? 1u : 0u) << (kt * 16 + g * 4 + r);
        }
      }
      const uint32_t vis = (visible_bits(k0, pos, a.window, a.sinks) & mbits) >> (4 * g);
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float sc = kCache && page < 0 ? __builtin_nanf("") : s[kt][r];
          s[kt][r] = seen_or_none(sc, vis, 16 * kt + r);
        }
      Finite v;
      bool dirty = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kCache) {
          dirty |= ((raw.vs[i >> 2] >> (8 * (i & 3))) & 255u) >= 253u;  // an element may be one
        } else {
#pragma unroll
          for (int j = 0; j < W / 2; ++j) {
            const uint32_t w = raw.v[i][j];
            v.look(w);
          }
        }
      }
      zero = __any(dirty || v.broken());
    }
    // ---- softmax ----
    float mt = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mt *= a.scale_log2;
    if (__any(mt > m_ref + kMoveRef)) {
      const float nr = fmaxf(m_ref, quad_max(mt));
      const float al = rescale(m_ref, nr);
      m_ref = nr;
      l *= al;
#pragma unroll
      for (int j = 0; j < W; ++j) oacc[j] *= al;
    }
    const float nm = m_ref == -__builtin_inff() ? 0.f : -m_ref;
    u32x4 pk;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[kt][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kt][r], a.scale_log2, nm));
        l += s[kt][r];
      }
      pk[2 * kt] = pack_bf16x2(s[kt][0], s[kt][1]);
      pk[2 * kt + 1] = pack_bf16x2(s[kt][2], s[kt][3]);
    }
    const bf16x8 pf = __builtin_bit_cast(bf16x8, pk);
    // ---- V rows of the lane's 8 keys, W dimensions each, in bf16 pairs ----
    uint32_t vr[8][W / 2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kCache) {
        const uint32_t e = (raw.vs[i >> 2] >> (8 * (i & 3))) & 255u;
        const float sc = __builtin_bit_cast(float, e << 23);
        if constexpr (D == 128) {
          const uint32_t c = raw.v[i >> 2][i & 3];
          const u32x4 x = __builtin_bit_cast(u32x4, dequant8(c, sc));
#pragma unroll
          for (int j = 0; j < 4; ++j) vr[i][j] = x[j];
        } else {
          const uint32_t c = raw.v[0][i >> 1];
          if (i & 1) {
            vr[i][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 2));
            vr[i][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 3));
          } else {
            vr[i][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0));
            vr[i][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1));
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) vr[i][j] = raw.v[i][j];
      }
    }
    // V^T operand of the block of dimensions W m + j, m < 16
    auto turn = [&](int j) {
      u32x4 vf;
#pragma unroll
      for (int tp = 0; tp < 4; ++tp)
        vf[tp] = __builtin_amdgcn_perm(vr[2 * tp + 1][j / 2], vr[2 * tp][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
      return vf;
    };
    if (zero) {
      // A key that a query does not see weighs 0, and 0 times an infinity or a NaN is a NaN: they go to the queries
      // that see them behind the loop, and count as zeros here.
      odd_v = true;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < W / 2; ++j) vr[i][j] = finite2(vr[i][j]);
    }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int j = 0; j < W; ++j)
      oacc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, turn(j)), pf, oacc[j], 0, 0, 0);
  };

  // (the next tile is on its way while this one is computed; two ahead took registers from a third workgroup on the CU:
  // a token over 131072 cached slots 34.8 us, so 33.9)
  Raw<D, kCache> next;
  int next_page = -1;
  if (mine > 0) load(next, 0, next_page);
  for (int it = 0; it < mine; ++it) {
    Raw<D, kCache> cur = next;
    const int page = next_page;
    if (it + 1 < mine) load(next, it + 1, next_page);
    compute(cur, it, page);
  }

  if (__builtin_expect(odd_v, 0)) {  // this lane's dimensions: 4 W g .. + 4 W - 1, O^T element (j, r) the one at W r + j
    for (int it = 0; it < mine; ++it) {
      const int k0 = tile_at(it) * kTile;
      uint32_t mbits = ~0u;
      if constexpr (!kCache) {
        if (a.mask) mbits = static_cast<uint32_t>(__ballot(a.mask[b * a.mask_sb + min(k0 + (lane & 31), a.limit - 1)] != 0.f));
      }
      if (mbits == 0 || (whole(k0) && mbits == ~0u)) continue;  // (whole tiles: the products have them)
      const uint8_t* sc = nullptr;
      if constexpr (kCache) {
        const int page = __builtin_amdgcn_readfirstlane(a.table[b * a.table_sb + (k0 >> a.page_shift)]);
        if (page < 0 || page >= a.num_pages) continue;
        sc = a.cache + page * a.page_stride + hk * a.head_stride +
             ((k0 & ((1 << a.page_shift) - 1)) / kTile) * kv4::tile_bytes(D) + 33 * D + 4 * W * g / 32 * 32;
      }
      for (uint32_t vis = visible_bits(k0, pos, a.window, a.sinks) & mbits; vis; vis &= vis - 1) {
        const int key = __builtin_ctz(vis);
        if constexpr (kCache) {
          if (sc[kv4::v_group(key) * 8 + kv4::v_unit(key)] >= 253)
#pragma unroll
            for (int j = 0; j < W; ++j) oacc[j] += __builtin_nanf("");
        } else {
          const uint16_t* const src = a.v + b * a.v_sb + hk * a.v_sh + static_cast<int64_t>(k0 + key) * a.v_ss + 4 * W * g;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < W; ++j) {
              const uint16_t w = src[W * r + j];
              if ((w & 0x7f80) == 0x7f80) oacc[j][r] += bf16_bits_to_f32(w);
            }
        }
      }
    }
  }

  // ---- merge the waves ----
  const float lsum = quad_sum(l);
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      floatx4 x = {oacc[j][r], oacc[j + 1][r], oacc[j + 2][r], oacc[j + 3][r]};
      // (a query past the limit sees slots that nobody can read)
      if (kCache && pos >= a.limit) x = floatx4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
      *reinterpret_cast<floatx4*>(&sm_o[wave][n16][4 * W * g + W * r + j]) = x;
    }
  if (g == 0) {
    sm_ml[wave][n16][0] = m_ref;
    sm_ml[wave][n16][1] = lsum;
  }
  __syncthreads();
  const int tid = static_cast<int>(threadIdx.x);
  const int mr = tid >> 4, md = (tid & 15) * W;  // the row and the first of W dimensions that this thread finishes
  if (mr >= rows) return;  // (and all threads past the first 256)
  float m = -__builtin_inff(), lt = 0.f, w[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) m = fmaxf(m, sm_ml[i][mr][0]);
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    w[i] = rescale(sm_ml[i][mr][0], m);
    lt = __builtin_fmaf(sm_ml[i][mr][1], w[i], lt);
  }
  float acc[W];
#pragma unroll
  for (int j = 0; j < W; j += 4) {
    floatx4 x = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NW; ++i) x += *reinterpret_cast<const floatx4*>(&sm_o[i][mr][md + j]) * w[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j + e] = x[e];
  }
  if (a.splits == 1) {
    const float inv = inverse_sum(lt);
    const int i = query_of(a, mr), h = hk * a.group + mr - i * a.group;
    uint32_t out[W / 2];
#pragma unroll
    for (int j = 0; j < W; j += 2) out[j / 2] = pack_bf16x2(acc[j] * inv, acc[j + 1] * inv);
    uint16_t* const dst = a.o + b * a.o_sb + i * a.o_ss + h * a.o_sh + md;
    if constexpr (W == 8)
      *reinterpret_cast<u32x4*>(dst) = u32x4{out[0], out[1], out[2], out[3]};
    else
      *reinterpret_cast<u32x2*>(dst) = u32x2{out[0], out[1]};
  } else {
    const int64_t item = ((static_cast<int64_t>(b) * a.hkv + hk) * a.splits + split) * kRowsBlock + mr;
    const int64_t items = static_cast<int64_t>(a.batch) * a.hkv * a.splits * kRowsBlock;
#pragma unroll
    for (int j = 0; j < W; j += 4)
      *reinterpret_cast<floatx4*>(a.part + item * D + md + j) = floatx4{acc[j], acc[j + 1], acc[j + 2], acc[j + 3]};
    if (md == 0) {
      a.part[items * D + item * 2] = m;
      a.part[items * D + item * 2 + 1] = lt;
    }
  }
}

// ---------------------------------------------------------------------------
// Many query rows: 32 (token, head) rows of a KV head's group a wave, and tiles of 32 keys that the workgroup brings into
// LDS once, NG of them a step: bf16 rows straight from memory (buffer_load ... lds, up to two slots ahead of the matrix
// work), codes of the cache through registers, as the bf16 values they stand for.  The NW waves are NW / NG blocks of 32
// rows times NG key groups, which take a tile of the step each and add up their states at the end.
//   S^T = K Q^T and O^T += V^T P^T with v_mfma_f32_32x32x16_bf16: a lane owns a query column, so maxima, sums and
//   rescaling stay in the lane and its partner (lane ^ 32), and P^T goes from accumulator to operand in place.
//   Both operands lie in LDS as rows, 16-byte pieces of row r exchanged by an XOR: K's by r mod the pieces of a row
//   (a lane reads one piece of its own key: 8 lanes cover 8 bank groups), V's by 2 (r mod 4) (ds_read_b64_tr_b16
//   gathers 4 keys of 16 dimensions, 32 bytes of each of 4 rows, into the V^T operand).
// Rows in (token, head) order keep the workgroup's windows together: 128 rows of 4 heads a group span 32 tokens, so
// a window of 1024 takes 34 tiles of which every wave needs 33.
// Bound: a step of 128 rows and 32 keys costs a CU 0.6 us with three workgroups on it, 0.2 of them matrix instructions at
// their peak rate, most of the rest the softmax's vector work (8192 tokens of 32/8 heads of 128, window 1024: 162 us, 0.80
// PFLOP/s of what is seen; 4096 causal tokens: 146 us, 0.94, where a loop of nothing but the reads and products of such
// tiles ends at 1.14); 1 us where a workgroup has the CU for itself: LDS reads, products and softmax in a chain.
// ---------------------------------------------------------------------------
template <int N>
__device__ __forceinline__ void vm_wait_barrier() {  // all but this wave's last N loads have arrived, everywhere
  static_assert(N == 0 || N == 2 || N == 4, "vmcnt immediate");
  if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

__device__ __forceinline__ float pair_max(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return __builtin_bit_cast(float, b0) + __builtin_bit_cast(float, b1);
}

// 16 bytes from base + offset of every lane to LDS, lane after lane (base: uniform).
__device__ __forceinline__ void load_lds16(const void* base, uint8_t* lds, int offset) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, offset, 0, 0, 0);
}

// The V^T operands of two 32-dimension blocks: rows 8 x .. 8 x + 7 of LDS through the transposing read, x < 4.  The
// reads and their wait are one block: beside builtins of these reads the compiler waits for every load into LDS that is
// still in flight.
template <int ROWB>
__device__ __forceinline__ void read_v(u32x2 (&v0)[2][2], u32x2 (&v1)[2][2], uint32_t at0, uint32_t at1) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%11\n\t"
      "ds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %9\n\t"
      "ds_read_b64_tr_b16 %5, %9 offset:%10\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%11\n\t"
      "ds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v0[0][0]), "=&v"(v0[0][1]), "=&v"(v0[1][0]), "=&v"(v0[1][1]), "=&v"(v1[0][0]), "=&v"(v1[0][1]),
        "=&v"(v1[1][0]), "=&v"(v1[1][1])
      : "v"(at0), "v"(at1), "n"(8 * ROWB), "n"(16 * ROWB), "n"(24 * ROWB)
      : "memory");
}

template <int D, int NG, bool kCache, bool kMask, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 2 : NG == 4 ? 1 : NG == 2 || (D == 128 && kCache) ? 2 : D == 64 ? 4 : 3)
void tile_attn_kernel(StreamArgs a) {  // (three workgroups a CU with a key mask, 3 registers in scratch: 8192 tokens 148 -> 136 us)
  constexpr int NQ = NW / NG, RB = 32 * NQ;
  constexpr int KCH = D / 16;      // MFMA steps over head_dim
  constexpr int DBLK = D / 32;     // 32-dimension blocks of O^T
  constexpr int PCS = D / 8;       // 16-byte pieces of a row
  constexpr int ROWB = 2 * D;      // bytes of a row
  constexpr int CH = 32 * ROWB / 1024;   // 1 KB chunks of a tile's K or V
  constexpr int CPW = CH / NQ;           // of them a wave loads: the waves of a key group bring its tile
  constexpr int TILEB = 2 * 32 * ROWB;   // K and V of a tile in LDS; a ring slot holds NG tiles, a step's
  constexpr int NS = kCache || NG > 1 ? 2 : 3;  // ring slots
  constexpr int OP = D + 8;              // pitch of O rows staged in LDS
  constexpr int RING = NS * NG * TILEB, STAGE = NW * 32 * OP * 2;
  static_assert(NG == 1 || NG == 2 || NG == 4, "key groups");
  static_assert(NW == kWaves || (NW == 8 && NG > 1), "waves");
  constexpr int EXCH = NG > 1 ? NW * (DBLK * 4 + 1) * 1024 : 0;  // states that the key groups exchange
  constexpr int LDS = RING > STAGE ? (RING > EXCH ? RING : EXCH) : (STAGE > EXCH ? STAGE : EXCH);
  __shared__ __attribute__((aligned(1024))) uint8_t ring[LDS];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int l32 = lane & 31, g = lane >> 5;
  const int wq = wave % NQ, kg = wave / NQ;  // the wave's block of 32 rows, and its share of the tiles

  // Work item: (batch, kv head, row tile, split).  Workgroup i runs on XCD i % 8: the items of a pair (batch, kv head),
  // which read the same keys, stay on one XCD, and the pairs go round the XCDs (sequences of a batch may differ in length:
  // 8 padded ones of 777 tokens and 24 heads of 64 took 31.8 us with a sequence to an XCD, 29.4 so); the last pairs,
  // fewer than 8, are cut into 8 runs of items.
  int id;
  {
    const int xcd = static_cast<int>(blockIdx.x % 8), k = static_cast<int>(blockIdx.x / 8);
    const int items = a.row_tiles * a.splits, pairs = a.batch * a.hkv, round = pairs / 8 * items;
    if (k < round) {
      const int turn = static_cast<int>(div_u32(static_cast<uint32_t>(k), a.d_items));
      id = k + (turn * 7 + xcd) * items;  // pair 8 turn + xcd, its item k - turn items
    } else {
      const int left = pairs % 8 * items, per = left / 8, more = left % 8;
      id = round * 8 + (k - round) + xcd * per + min(xcd, more);
    }
  }
  const int split = split_off(id, a.splits, a.d_splits);
  const int rt = a.row_tiles - 1 - split_off(id, a.row_tiles, a.d_row_tiles);  // (the last rows first: they may have the longest spans)
  const int hk = split_off(id, a.hkv, a.d_hkv), b = id;

  const int rows = a.sq * a.group;
  const int row0 = rt * RB, rw0 = row0 + 32 * wq;
  const Span sp = span_of<kCache>(a, b, row0, min(RB, rows - row0));
  const int use = splits_of(a.splits, sp.n);
  if (split >= use) return;
  const int t0 = split_start(sp.n, split, use), n = split_start(sp.n, split + 1, use) - t0;
  auto tile_at = [&](int it) {
    const int t = t0 + min(it, n - 1);  // (past the end: the last one again)
    return t < sp.ns ? t : sp.w0 + (t - sp.ns);
  };

  // this lane's query, and the first and last slot of the wave's queries
  const int row = min(rw0 + l32, rows - 1);
  const int qi = query_of(a, row), qh = hk * a.group + row - qi * a.group;
  const int pos = qi < sp.count ? max(sp.start + qi, -1) : -1;
  const int pw0 = sp.start + query_of(a, rw0), pw1 = sp.start + query_of(a, min(rw0 + 32, rows) - 1);
  // (every query of the wave sees something)
  const bool all_rows = rw0 < rows && pw0 >= 0 && pw0 >= sp.p0 && pw1 <= sp.p1;
  bf16x8 qf[KCH];
  {
    const uint16_t* const src = a.q + b * a.q_sb + qi * a.q_ss + qh * a.q_sh + 8 * g;
#pragma unroll
    for (int ks = 0; ks < KCH; ++ks) qf[ks] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(src + 16 * ks));
  }

  // ---- tiles into LDS ----
  const uint16_t* const kb = kCache ? nullptr : a.k + b * a.k_sb + hk * a.k_sh;
  const uint16_t* const vb = kCache ? nullptr : a.v + b * a.v_sb + hk * a.v_sh;
  auto swz_k = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
  auto swz_v = [](int r) { return D == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); };
  // this lane's rows and pieces of the wave's chunks
  int drow[CPW], dk[CPW], dv[CPW];
#pragma unroll
  for (int c = 0; c < CPW; ++c) {
    drow[c] = (wq + NQ * c) * (1024 / ROWB) + lane / PCS;
    dk[c] = drow[c] * static_cast<int>(a.k_ss * 2) + ((lane % PCS) ^ swz_k(drow[c])) * 16;
    dv[c] = drow[c] * static_cast<int>(a.v_ss * 2) + ((lane % PCS) ^ swz_v(drow[c])) * 16;
  }
  // the next tile that the workgroup brings: its first key and its rows (past the end: the last one again)
  const int64_t kstep = a.k_ss * (2 * kTile), vstep = a.v_ss * (2 * kTile);
  const uint8_t *kt = nullptr, *vt = nullptr;
  int d_it = 0, d_tile = 0;
  auto dma_seek = [&](int tile) {
    d_tile = tile;
    kt = reinterpret_cast<const uint8_t*>(kb) + tile * kstep;
    vt = reinterpret_cast<const uint8_t*>(vb) + tile * vstep;
  };
  auto dma = [&](int off) {
    const int k0 = d_tile * kTile;
    uint8_t* const to = ring + off + wq * 1024;
    int ok[CPW], ov[CPW];
#pragma unroll
    for (int c = 0; c < CPW; ++c) ok[c] = dk[c], ov[c] = dv[c];
    if (k0 + kTile > a.limit) {  // rows past the last key repeat it
#pragma unroll
      for (int c = 0; c < CPW; ++c) {
        const int past = max(drow[c] - (a.limit - 1 - k0), 0);
        ok[c] -= past * static_cast<int>(a.k_ss * 2);
        ov[c] -= past * static_cast<int>(a.v_ss * 2);
      }
    }
#pragma unroll
    for (int c = 0; c < CPW; ++c) load_lds16(kt, to + NQ * c * 1024, ok[c]);
#pragma unroll
    for (int c = 0; c < CPW; ++c) load_lds16(vt, to + 32 * ROWB + NQ * c * 1024, ov[c]);
    if constexpr (NG > 1) {
      d_it += NG;
      dma_seek(tile_at(d_it));
    } else if (++d_it < n) {
      if (d_tile + 1 == sp.ns) {
        dma_seek(sp.w0);
      } else {
        ++d_tile;
        kt += kstep;
        vt += vstep;
      }
    }
  };
  // page ids of 64 tiles, one a lane
  int ids = -1, ids_base = 0;
  auto load_ids = [&](int it0) {
    ids_base = it0;
    ids = -1;
    if constexpr (kCache) {
      const int it = it0 + lane;
      if (it < n) ids = a.table[b * a.table_sb + ((tile_at(it) * kTile) >> a.page_shift)];
    }
  };
  auto page_of = [&](int it) {  // called with it ascending
    if (it - ids_base >= 64) load_ids(it);
    const int page = __builtin_amdgcn_readlane(ids, it - ids_base);
    return page < a.num_pages ? max(page, -1) : -1;
  };
  auto tile_ptr = [&](int page, int it) {
    return a.cache + page * a.page_stride + hk * a.head_stride +
           (((tile_at(it) * kTile) & ((1 << a.page_shift) - 1)) / kTile) * kv4::tile_bytes(D);
  };
  // A tile in 256 shares, 64 a wave at a time: part 0 and 1 are K's, D / 4 dimensions of a row each, 2 and 3 V's, half of a
  // lane's units (16 lanes next to each other: what they write at once lies in different banks).
  auto fetch = [&](int page, int it, int part, u32x4& codes, uint32_t& scales) {
    codes = u32x4{0, 0, 0, 0};
    scales = 0;
    if (page < 0) return;
    const uint8_t* const t = tile_ptr(page, it);
    const int ct = (part & 1) * 64 + lane, half = ct >> 4 & 1, lb = ct >> 5 << 4 | (ct & 15);
    const uint8_t* const src = t + (part < 2 ? ct * (D / 8) : 16 * D + (2 * lb + half) * (D / 8));
    if constexpr (D == 128) {
      codes = *reinterpret_cast<const u32x4*>(src);
    } else {
      const u32x2 x = *reinterpret_cast<const u32x2*>(src);
      codes = u32x4{x[0], x[1], 0, 0};
    }
    if (part < 2) {
      scales = t[32 * D + (ct >> 2) * (D / 32) + (D == 128 ? ct & 3 : (ct & 3) >> 1)];
    } else {  // the scales of 4 slots
      scales = *reinterpret_cast<const uint32_t*>(t + 33 * D + ((lb & 15) * (D / 16) / 32 * 4 + (lb >> 4)) * 8 + half * 4);
    }
  };
  auto store = [&](int off, int part, u32x4 codes, uint32_t scales) {
    uint8_t* const ks = ring + off;
    const int ct = (part & 1) * 64 + lane;
    if (part < 2) {
      const int r = ct >> 2;
      const float sc = __builtin_bit_cast(float, scales << 23);
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint32_t c = codes[j];
        const int piece = (ct & 3) * (D / 32) + j;
        *reinterpret_cast<bf16x8*>(ks + r * ROWB + (piece ^ swz_k(r)) * 16) = dequant8(c, sc);
      }
    } else {
      const int r0 = 16 * (ct >> 4 & 1) + 4 * (ct >> 5), col = ct & 15;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + j;
        const float sc = __builtin_bit_cast(float, ((scales >> (8 * j)) & 255u) << 23);
        uint8_t* const dst = ks + 32 * ROWB + r * ROWB;
        if constexpr (D == 128) {
          const uint32_t c = codes[j];
          *reinterpret_cast<bf16x8*>(dst + (col ^ swz_v(r)) * 16) = dequant8(c, sc);
        } else {
          uint32_t c = codes[j >> 1];
          c = j & 1 ? c >> 16 : c;
          const u32x2 x = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 0)),
                           __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, sc, 1))};
          *reinterpret_cast<u32x2*>(dst + ((col >> 1) ^ swz_v(r)) * 16 + (col & 1) * 8) = x;
        }
      }
    }
  };

  floatx16 oacc[DBLK];
#pragma unroll
  for (int db = 0; db < DBLK; ++db) oacc[db] = floatx16{};
  // The softmax reference m_ref (log2 units), the score beyond which it moves, and -m_ref for the exponent's argument
  // (0 as long as there is none: p = exp2(-inf) = 0)
  float m_ref = -__builtin_inff(), m_move = -__builtin_inff(), m_neg = 0.f, l = 0.f;

  // the mask of a tile's keys, a bit each (lanes 0 .. 31 load them, a step ahead)
  float mload = 1.f;
  auto fetch_mask = [&](int it) {
    if constexpr (kMask) mload = a.mask[b * a.mask_sb + min(tile_at(it) * kTile + l32, a.limit - 1)];
  };

  // LDS addresses of this lane's part of the operands: piece g of row l32 of K; 8 bytes of row 4 g + (lane / 4) % 4 of
  // every 8 rows of V (piece 2 (lane / 16 % 2) + lane / 2 % 2)
  const uint32_t ring_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)ring));
  const uint32_t k_at = ring_at + l32 * ROWB + (g ^ swz_k(l32)) * 16;
  const uint32_t v_at = ring_at + 32 * ROWB + (4 * g + ((lane >> 2) & 3)) * ROWB + (lane & 1) * 8 +
                        ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ swz_v(lane >> 2)) * 16;

  auto skipped = [&](int k0) { return k0 > pw1 || (k0 + kTile - 1 <= pw0 - a.window && k0 >= a.sinks) || rw0 >= rows; };
  // every query of the wave sees all 32 keys
  auto whole = [&](int k0) {
    const bool low = k0 > pw1 - a.window, sink = k0 + kTile <= a.sinks, high = k0 + kTile - 1 <= pw0;
    return all_rows & high & (low | sink);
  };
  auto load_k = [&](u32x4 (&kop)[KCH], int off) {
    // (piece 2 c + g is the swizzled piece g with 2 c exchanged too: one address and an XOR for each)
    const uint32_t at = k_at + off;
#pragma unroll
    for (int c = 0; c < KCH; ++c)
      kop[c] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4*>(at ^ (32 * c));
  };
  auto load_v = [&](u32x2 (&vop)[DBLK][2][2], int off) {
    const uint32_t at = v_at + off;
#pragma unroll
    for (int db = 0; db < DBLK; db += 2) read_v<ROWB>(vop[db], vop[db + 1], at ^ (64 * db), at ^ (64 * db + 64));
  };
  auto top_of = [&](const floatx16& s) {
    float mt = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mt = fmaxf(mt, s[e]);
    return mt;
  };
  const float inv_scale = 1.f / a.scale_log2;
  auto move_ref = [&](float mt) {
    const float nr = fmaxf(m_ref, pair_max(mt) * a.scale_log2);
    const float al = rescale(m_ref, nr);
    m_ref = nr;
    m_move = (nr + kMoveRef) * inv_scale;
    m_neg = nr == -__builtin_inff() ? 0.f : -nr;
    l *= al;
#pragma unroll
    for (int db = 0; db < DBLK; ++db) oacc[db] *= al;
  };
  auto exp_all = [&](floatx16& s) {
    float ps = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], a.scale_log2, m_neg));
      ps += s[e];
    }
    l += ps;
  };
  auto pack = [&](const floatx16& s, u32x4 (&pk)[2]) {
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
      pk[s2] = u32x4{pack_bf16x2(s[8 * s2], s[8 * s2 + 1]), pack_bf16x2(s[8 * s2 + 2], s[8 * s2 + 3]),
                     pack_bf16x2(s[8 * s2 + 4], s[8 * s2 + 5]), pack_bf16x2(s[8 * s2 + 6], s[8 * s2 + 7])};
  };
  auto pv = [&](const u32x2 (&vop)[DBLK][2][2], const u32x4 (&pk)[2]) {
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int db = 0; db < DBLK; ++db) {
        const u32x4 vf = {vop[db][s2][0][0], vop[db][s2][0][1], vop[db][s2][1][0], vop[db][s2][1][1]};
        oacc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf), __builtin_bit_cast(bf16x8, pk[s2]),
                                                           oacc[db], 0, 0, 0);
      }
  };
  bool odd_v = false;  // (wave-uniform) some tile's V held infinities or NaN that not every query of the wave sees

  // Any tile.
  // Tiles that start at w_lo .. w_lo + w_len - 1 lie whole in the windows of all of the wave's queries.
  const int w_lo = max(pw1 - a.window + 1, 0), w_len = all_rows ? max(pw0 - kTile + 2 - w_lo, 0) : 0;
  auto compute = [&](int k0, int off, int page, uint32_t mbits) {
    bool full = static_cast<unsigned>(k0 - w_lo) < static_cast<unsigned>(w_len);
    if (!full) {
      if (skipped(k0)) return;
      full = whole(k0);  // (the sinks' tiles)
    }
    if (kMask && mbits == 0) return;
    full = full && page >= 0 && mbits == 0xffffffffu;
    floatx16 s = floatx16{};
    u32x2 vop[DBLK][2][2];
    {
      u32x4 kop[KCH];
      load_k(kop, off);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < KCH; ++c)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kop[c]), qf[c], s, 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_v(vop, off);
    __builtin_amdgcn_sched_barrier(0);
    // ---- visibility ----
    if (!full) {
      const uint32_t vis = (visible_bits(k0, pos, a.window, a.sinks) & mbits) >> (4 * g);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float sc = kCache && page < 0 ? __builtin_nanf("") : s[e];
        s[e] = seen_or_none(sc, vis, 8 * (e >> 2) + (e & 3));
      }
      Finite v;
#pragma unroll
      for (int db = 0; db < DBLK; ++db)
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < 2; ++x) v.look(vop[db][s2][h][x]);
      if (__any(v.broken())) {
        // A key that a query does not see weighs 0, and 0 times an infinity or a NaN is a NaN: they go to the queries
        // that see them behind the loop, and count as zeros here.
        odd_v = true;
#pragma unroll
        for (int db = 0; db < DBLK; ++db)
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int x = 0; x < 2; ++x) vop[db][s2][h][x] = finite2(vop[db][s2][h][x]);
      }
    }
    const float mt = top_of(s);
    if (__any(mt > m_move)) move_ref(mt);
    u32x4 pk[2];
    exp_all(s);
    pack(s, pk);
    pv(vop, pk);
  };

  if (n > 0) {
    // step st brings the tiles st NG .. + NG - 1, of which key group kg takes st NG + kg
    const int steps = (n + NG - 1) / NG;
    if constexpr (kCache) {
      load_ids(0);
      constexpr int PARTS = 4 / NQ;  // of its key group's tile a wave takes
      u32x4 codes[PARTS];
      uint32_t scales[PARTS];
      int own = -1, own_next = -1;  // the page of this wave's tile
      auto fetch_step = [&](int st) {
        const int page = st * NG + kg < n ? page_of(st * NG + kg) : -1;
#pragma unroll
        for (int x = 0; x < PARTS; ++x) fetch(page, st * NG + kg, wq + NQ * x, codes[x], scales[x]);
        return page;
      };
      auto store_step = [&](int slot) {
#pragma unroll
        for (int x = 0; x < PARTS; ++x) store((slot * NG + kg) * TILEB, wq + NQ * x, codes[x], scales[x]);
      };
      own = fetch_step(0);
      store_step(0);
      if (steps > 1) own_next = fetch_step(1);
      for (int st = 0; st < steps; ++st) {
        if constexpr (NQ == 1)  // (a tile of one wave's own: what it wrote and read it has waited for itself)
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        else
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int page = own;
        own = own_next;
        if (st + 1 < steps) store_step((st + 1) & 1);
        if (st + 2 < steps) own_next = fetch_step(st + 2);
        if (st * NG + kg < n) compute(tile_at(st * NG + kg) * kTile, ((st & 1) * NG + kg) * TILEB, page, ~0u);
      }
    } else {
      auto dma_step = [&](int slot) { dma((slot * NG + kg) * TILEB); };
      fetch_mask(kg);
      d_it = kg;
      dma_seek(tile_at(d_it));
#pragma unroll
      for (int x = 0; x < NS - 1; ++x) dma_step(x);
      int slot = 0, into = NS - 1;
      for (int st = 0; st < steps; ++st) {
        if constexpr (NQ == 1)  // (a tile of one wave's own)
          asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else
          vm_wait_barrier<(NS - 2) * 2 * CPW>();  // the step's tiles are in LDS, the slot of the last step is free
        uint32_t mask = ~0u;
        if constexpr (kMask) mask = static_cast<uint32_t>(__ballot(mload != 0.f));
        fetch_mask((st + 1) * NG + kg);
        dma_step(into);
        if (st * NG + kg < n) compute(tile_at(st * NG + kg) * kTile, (slot * NG + kg) * TILEB, 0, mask);
        into = slot;
        slot = slot + 1 == NS ? 0 : slot + 1;
      }
    }
  }
  vm_wait_barrier<0>();  // every wave has read its last tile, no load into LDS is in flight

  if (__builtin_expect(odd_v, 0)) {
    for (int it = kg; it < n; it += NG) {
      const int k0 = tile_at(it) * kTile;
      if (skipped(k0)) continue;
      uint32_t mbits = ~0u;
      if constexpr (kMask) mbits = static_cast<uint32_t>(__ballot(a.mask[b * a.mask_sb + min(k0 + l32, a.limit - 1)] != 0.f));
      if (mbits == 0 || (whole(k0) && mbits == ~0u)) continue;  // (whole tiles: the products have them)
      uint32_t vis = visible_bits(k0, pos, a.window, a.sinks) & mbits;
      if constexpr (kCache) {
        const int page = __builtin_amdgcn_readfirstlane(a.table[b * a.table_sb + (k0 >> a.page_shift)]);
        if (page < 0 || page >= a.num_pages) continue;
        const uint8_t* const sc = tile_ptr(page, it) + 33 * D;
        for (; vis; vis &= vis - 1) {
          const int key = __builtin_ctz(vis);
#pragma unroll
          for (int db = 0; db < DBLK; ++db)
            if (sc[(db * 4 + kv4::v_group(key)) * 8 + kv4::v_unit(key)] >= 253) oacc[db] += __builtin_nanf("");
        }
      } else {
        for (; vis; vis &= vis - 1) {
          const uint16_t* const src = vb + static_cast<int64_t>(k0 + __builtin_ctz(vis)) * a.v_ss + 4 * g;
#pragma unroll
          for (int db = 0; db < DBLK; ++db)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const uint16_t w = src[32 * db + 8 * (x >> 2) + (x & 3)];
              if ((w & 0x7f80) == 0x7f80) oacc[db][x] += bf16_bits_to_f32(w);
            }
        }
      }
    }
  }

  float lt = pair_sum(l);
  const int row_at = rw0 + l32;
  if constexpr (NG > 1) {
    // The key groups of a row block exchange their states; group kg finishes the blocks kg, kg + NG, ... of O^T.
    floatx4* const ex = reinterpret_cast<floatx4*>(ring);
    constexpr int PER = (DBLK * 4 + 1) * 64;
    floatx4* const mine = ex + wave * PER;
#pragma unroll
    for (int db = 0; db < DBLK; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        mine[(db * 4 + q4) * 64 + lane] = floatx4{oacc[db][4 * q4], oacc[db][4 * q4 + 1], oacc[db][4 * q4 + 2], oacc[db][4 * q4 + 3]};
    mine[DBLK * 4 * 64 + lane] = floatx4{m_ref, lt, 0.f, 0.f};
    __syncthreads();
    float mg[NG], wg[NG], m = -__builtin_inff();
    lt = 0.f;
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      mg[x] = ex[(wq + NQ * x) * PER + DBLK * 4 * 64 + lane][0];
      m = fmaxf(m, mg[x]);
    }
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      wg[x] = rescale(mg[x], m);
      lt = __builtin_fmaf(ex[(wq + NQ * x) * PER + DBLK * 4 * 64 + lane][1], wg[x], lt);
    }
    m_ref = m;
#pragma unroll
    for (int y = 0; y < (DBLK + NG - 1) / NG; ++y) {
      const int db = kg + y * NG;
      if (db < DBLK) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          floatx4 x = {0, 0, 0, 0};
#pragma unroll
          for (int z = 0; z < NG; ++z) x += ex[(wq + NQ * z) * PER + (db * 4 + q4) * 64 + lane] * wg[z];
#pragma unroll
          for (int e = 0; e < 4; ++e) oacc[y][4 * q4 + e] = x[e];
        }
      }
    }
  }
  constexpr int MINE = (DBLK + NG - 1) / NG;  // blocks of O^T that this wave finishes, the y-th at kg + y NG
  if (a.splits > 1) {
    // Whole lines of 128 bytes, 32 dimensions of a row by 8 lanes, through LDS, and past the L2: what is left there has to
    // leave it before the merge begins.  2 x 49 tokens of 28/4 heads of 128 over 6000 slots, 16 MB of states: 31.8 us with
    // 16-byte pieces that stay in the L2, 29.7 so.
    constexpr int PITCH = 36;  // floats of a row's 32 in LDS
    static_assert(NW * 32 * PITCH * 4 <= LDS, "states in LDS");
    const int64_t item0 = (((static_cast<int64_t>(b) * a.hkv + hk) * a.row_tiles + rt) * a.splits + split) * RB + 32 * wq;
    const int64_t items = static_cast<int64_t>(a.batch) * a.hkv * a.row_tiles * a.splits * RB;
    __syncthreads();  // (the other key groups have read this wave's state)
    float* const rows32 = reinterpret_cast<float*>(ring) + wave * (32 * PITCH);
#pragma unroll
    for (int y = 0; y < MINE; ++y)
      if (kg + y * NG < DBLK) {
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          floatx4 x = {oacc[y][4 * q4], oacc[y][4 * q4 + 1], oacc[y][4 * q4 + 2], oacc[y][4 * q4 + 3]};
          if (kCache && pos >= a.limit) x = floatx4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
          *reinterpret_cast<floatx4*>(rows32 + l32 * PITCH + 8 * q4 + 4 * g) = x;
        }
#pragma unroll
        for (int z = 0; z < 4; ++z) {  // (a wave reads what it wrote itself)
          const int r = 8 * z + lane / 8;
          const floatx4 x = *reinterpret_cast<const floatx4*>(rows32 + r * PITCH + lane % 8 * 4);
          if (rw0 + r < rows)
            __builtin_nontemporal_store(x, reinterpret_cast<floatx4*>(a.part + (item0 + r) * D + 32 * (kg + y * NG) + lane % 8 * 4));
        }
      }
    if (g == 0 && kg == 0 && row_at < rows) {
      a.part[items * D + (item0 + l32) * 2] = m_ref;
      a.part[items * D + (item0 + l32) * 2 + 1] = lt;
    }
    return;
  }
  float inv = inverse_sum(lt);
  if (kCache && pos >= a.limit) inv = __builtin_nanf("");  // (sees slots that nobody can read)
  if constexpr (NG > 1) {
    if (row_at < rows) {
      uint16_t* const dst = a.o + b * a.o_sb + qi * a.o_ss + qh * a.o_sh + 4 * g;
#pragma unroll
      for (int y = 0; y < MINE; ++y)
        if (kg + y * NG < DBLK) {
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4)
            *reinterpret_cast<u32x2*>(dst + 32 * (kg + y * NG) + 8 * q4) =
                u32x2{pack_bf16x2(oacc[y][4 * q4] * inv, oacc[y][4 * q4 + 1] * inv),
                      pack_bf16x2(oacc[y][4 * q4 + 2] * inv, oacc[y][4 * q4 + 3] * inv)};
        }
    }
    return;
  }
  uint16_t* const st = reinterpret_cast<uint16_t*>(ring) + wave * (32 * OP);
#pragma unroll
  for (int db = 0; db < DBLK; ++db)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4)
      *reinterpret_cast<u32x2*>(st + l32 * OP + 32 * db + 8 * q4 + 4 * g) =
          u32x2{pack_bf16x2(oacc[db][4 * q4] * inv, oacc[db][4 * q4 + 1] * inv),
                pack_bf16x2(oacc[db][4 * q4 + 2] * inv, oacc[db][4 * q4 + 3] * inv)};
  // whole rows in 16-byte pieces (a wave reads what it wrote itself), past the L2: 1280 tokens of 28/4 heads of 128 27.1 ->
  // 26.4 us, 8 x 777 of 24 of 64 29.9 -> 28.7
#pragma unroll
  for (int x = 0; x < 32 * PCS / 64; ++x) {
    const int r = x * (64 / PCS) + lane / PCS, c = lane % PCS * 8;
    const u32x4 w = *reinterpret_cast<const u32x4*>(st + r * OP + c);
    const int orow = rw0 + r;
    if (orow >= rows) continue;
    const int i = query_of(a, orow), h = hk * a.group + orow - i * a.group;
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(a.o + b * a.o_sb + i * a.o_ss + h * a.o_sh + c));
  }
}

// x of the lane y further round in this lane's 16
__device__ __forceinline__ float row_turned(float x, int y) {
  const int b = __builtin_bit_cast(int, x);
  const int r = y == 1 ? __builtin_amdgcn_mov_dpp(b, 0x121, 0xf, 0xf, false)
              : y == 2 ? __builtin_amdgcn_mov_dpp(b, 0x122, 0xf, 0xf, false)
              : y == 4 ? __builtin_amdgcn_mov_dpp(b, 0x124, 0xf, 0xf, false)
                       : __builtin_amdgcn_mov_dpp(b, 0x128, 0xf, 0xf, false);
  return __builtin_bit_cast(float, r);
}

// O of the query rows from the partial states of their splits: `per` waves (1 up to 16 splits, else 4) to a row, wave w
// of them adds up splits w, w + per, ... .  Every state is loaded before anything is known about its use: one round trip
// through memory, whichever of the splits had tiles.
template <int D, bool kCache>
__global__ __launch_bounds__(64 * kWaves) void merge_kernel(StreamArgs a, int rb, int per) {
  constexpr int E = D / 64;  // dimensions per lane
  constexpr int U = kMaxSplits / kWaves;
  __shared__ float sm[kWaves][D];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int rows = a.sq * a.group, share = wave % per;
  const int at = static_cast<int>(blockIdx.x) * (kWaves / per) + wave / per;
  if (at >= a.batch * a.hkv * rows) return;  // (one wave to a row: no barrier follows)
  const int bh = at / rows, row = at - bh * rows;
  const int b = bh / a.hkv, hk = bh - b * a.hkv;
  const int rt = row / rb;
  const int64_t first = (static_cast<int64_t>(bh) * a.row_tiles + rt) * a.splits * rb + (row - rt * rb);
  const int64_t items = static_cast<int64_t>(a.batch) * a.hkv * a.row_tiles * a.splits * rb;
  float x[U][E] = {};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s = share + per * u;
    if (s < a.splits) {
      const float* const src = a.part + (first + static_cast<int64_t>(s) * rb) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = src[e];
    }
  }
  float m = -__builtin_inff(), l = 0.f;
  if (lane < a.splits) {
    const float* const ml = a.part + items * D + (first + static_cast<int64_t>(lane) * rb) * 2;
    m = ml[0];
    l = ml[1];
  }
  const Span sp = span_of<kCache>(a, b, rt * rb, min(rb, rows - rt * rb));
  const int use = splits_of(a.splits, sp.n);
  m = lane < use ? m : -__builtin_inff();
  float top = m;
#pragma unroll
  for (int y = 1; y < 16; y *= 2) top = fmaxf(top, row_turned(top, y));
  top = quad_max(top);
  const float w = rescale(m, top);
  l = lane < use ? l * w : 0.f;
#pragma unroll
  for (int y = 1; y < 16; y *= 2) l += row_turned(l, y);
  l = quad_sum(l);
  float acc[E] = {};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int s = share + per * u;
    if (s < use) {
      const float ws = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s));
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(x[u][e], ws, acc[e]);
    }
  }
  if (per > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) sm[wave][lane * E + e] = acc[e];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[e] = sm[0][lane * E + e];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) acc[e] += sm[i][lane * E + e];
    }
  }
  const float inv = inverse_sum(l);
  const int i = query_of(a, row), h = hk * a.group + row - i * a.group;
  uint16_t* const dst = a.o + b * a.o_sb + i * a.o_ss + h * a.o_sh + lane * E;
  if constexpr (E == 2)
    *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  else
    *dst = f32_to_bf16_bits(acc[0] * inv);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
bool a16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How a call is cut up; depends on sizes alone.
struct Plan {
  int waves;                  // of a workgroup: 4 or 8
  int rb, row_tiles, splits;  // rows of a workgroup: 16 (rows_attn_kernel), 32, 64 or 128 (tile_attn_kernel)
  int64_t items;              // row blocks times splits
  int64_t workspace(int64_t head_dim) const { return splits > 1 ? items * rb * (head_dim + 2) * 4 : 0; }
};

// limit: readable keys.  false: sizes that the kernels do not take.
bool plan_of(Plan& p, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t seq_q, int64_t limit, int64_t head_dim,
             int64_t window, int64_t sinks, bool cache) {
  if ((head_dim != 64 && head_dim != 128) || batch < 0 || q_heads < 0 || kv_heads <= 0 || q_heads % kv_heads ||
      seq_q < 0 || limit < 0 || limit > kMaxSlots || window < 1 || sinks < 0 || batch > 65535 || q_heads > 65535 ||
      kv_heads > 65535)
    return false;
  const int64_t group = q_heads / kv_heads, rows = seq_q * group;
  if (seq_q > kMaxSlots || rows > kMaxSlots) return false;
  const int64_t heads = std::max<int64_t>(1, batch * kv_heads);
  // workgroups of 32 (bf16 rows; twice as many of 64) or 128 rows (codes, 8 waves) that a CU's LDS holds
  const int64_t cus = 256, per_cu = head_dim == 128 ? 1 : 2;
  const auto row_tiles = [&](int64_t rb) { return std::max<int64_t>(1, (rows + rb - 1) / rb); };
  // tiles of the longest block of rb rows
  const auto tiles_of = [&](int64_t rb) {
    const int64_t span = std::min(limit, std::min(window, limit) + rb / std::max<int64_t>(1, group) + 1);
    return std::min((limit + kTile - 1) / kTile,
                    (std::min(sinks, limit) + kTile - 1) / kTile + (span + kTile - 1) / kTile + 1);
  };
  const auto splits_for = [&](int64_t blocks, int64_t tiles, int64_t workgroups) {
    return std::min<int64_t>({kMaxSplits, std::max<int64_t>(1, workgroups / blocks), std::max<int64_t>(1, (tiles + kWaves - 1) / kWaves)});
  };
  // steps that a CU takes, one after the other, over blocks of rb rows and `per` tiles a step
  const auto steps_of = [&](int64_t rb, int64_t per) {
    const int64_t blocks = heads * row_tiles(rb), tiles = tiles_of(rb), splits = splits_for(blocks, tiles, cus);
    return ((tiles + splits - 1) / splits + per - 1) / per * ((blocks * splits + cus - 1) / cus);
  };
  p.waves = 4;
  if (rows <= kRowsBlock) {
    p.rb = kRowsBlock;
  } else if (cache) {
    // Every row block turns the codes into values again, 32 rows 4 times as often as 128, but the fewer rows, the more
    // keys a step takes (4 tiles, 2 of 128 rows) and the fewer partial states leave the chip.  A step takes 2 us (32 rows,
    // 4 waves; 64 rows, 8 waves), 1.3 (128 rows, 8 waves).  us for 32 / 64 / 128 rows, head_dim 128: 49 tokens of 28/4
    // heads over 300 slots 11.6 / 13.1 / 14.1, over 6000 25.2 / 22.1 / 25.1, 2 sequences of them 42 / 29 / 30;
    // 169 tokens over 500 slots 11.3 / 17.7 / 18.4, over 2000 27 / 23 / 26, over 20000 210 / 97 / 86.  64 rows as well
    // where their blocks fill the chip without shares of the keys: 512 tokens of 32/8 heads over 4096 slots 90 / 58 / 64,
    // of 64 43 / 41 / 46, 700 over 2000 37 / 29 / 43.
    const int64_t blocks64 = heads * row_tiles(64);
    p.rb = steps_of(32, 4) <= 4 ? 32 : steps_of(64, 4) <= 8 || (blocks64 >= cus * 7 / 8 && blocks64 <= per_cu * cus) ? 64 : 128;
    // Blocks of 128 rows that do not run at once: 4 waves, a tile a step (4096 tokens of 32/8 heads over 8192 slots 471
    // us, 516 with 8 waves; 1024 tokens, which do, 246 and 172).
    if (p.rb == 64 || (p.rb == 128 && heads * row_tiles(128) <= per_cu * cus)) p.waves = 8;
  } else {
    // The smallest row blocks whose workgroups run all at once, else 128 rows by 4 waves (us for 32 / 64 / 128 rows of 28/4
    // heads of 128: 169 queries over 1449 keys 14 / 19 / 22, 640 x 640, window 512, 23 / 16 / 21, 1280 x 1280 44 / 31 / 26).
    // But each block reads its keys again, and few blocks share them out: over long ranges 64 rows, then 128 by 8 waves, two
    // tiles a step (32 / 64 / these: 169 x 3000 25 / 26 / 26, 169 x 8192 54 / 46 / 35, 300 x 8192 104 / 103 / 56; 300 x 1449
    // 25 / 20 / 25).  head_dim 64 with two workgroups of 32 rows on most CUs: 512 x 4096 of 32/8 heads 30 / 39 / 40.
    const int64_t blocks32 = heads * row_tiles(32), blocks64 = heads * row_tiles(64), steps32 = steps_of(32, 4);
    if (blocks32 <= per_cu * cus && (steps32 <= 16 || (blocks32 > cus && steps32 <= 64)))
      p.rb = 32;
    else if (blocks64 <= 2 * per_cu * cus && !(blocks64 <= cus && steps_of(64, 2) > 20))
      p.rb = 64;
    else
      p.rb = 128;
    if (p.rb == 128 && blocks64 <= cus) p.waves = 8;
  }
  p.row_tiles = static_cast<int>(row_tiles(p.rb));
  const int64_t blocks = heads * p.row_tiles, tiles = tiles_of(p.rb);
  p.splits = static_cast<int>(splits_for(blocks, tiles, (p.rb == kRowsBlock ? 2 : 1) * cus));
  // (two workgroups of 8 waves to a CU, of head_dim 64, where each has tiles enough: 169 tokens of 28/4 heads over 20000 slots
  // 63 -> 53 us, 300 over 8192 keys 43 -> 37; 2 x 49 over 6000 slots, 19 tiles each, 22 -> 27)
  if (p.rb == 128 && p.waves == 8 && head_dim == 64 && tiles >= 40 * p.splits)
    p.splits = static_cast<int>(splits_for(blocks, tiles, 2 * cus));
  // Sharing a row block out means a second launch, about 3 us.  Where 8 waves walk the tiles in (nearly) as few steps as
  // 4 waves of each split do, one workgroup of 8 takes the row block whole.  A step takes a workgroup 0.5 us (codes,
  // head_dim 64), 0.9 (codes, or rows of 64) or 1.7 (rows of 128, 128 KB).  Token of 32/8 heads of 128, shared out ->
  // whole: 250 slots 7.4 -> 4.9, 1500 slots 7.7 (10.1 whole), 32 sequences of 1500 slots 16.1 -> 12.7; bf16 rows: 250 keys
  // 7.9 -> 6.1, 500 keys 7.9 (8.6 whole), 32 sequences of 1000 keys 29.3 -> 25.9.
  if (p.rb == kRowsBlock && p.splits > 1) {
    const int64_t more = (tiles + 7) / 8 - (tiles + 4 * p.splits - 1) / (4 * p.splits);
    if (more <= (!cache && head_dim == 128 ? 0 : 2))
      p.waves = 8, p.splits = 1;
    else if (head_dim == 64)  // three workgroups of 4 waves on a CU: 16 x 8000 keys of 24/8 heads 59 -> 54 us, slots 20.3 -> 19.4
      p.splits = static_cast<int>(splits_for(blocks, tiles, 3 * cus));
  }
  p.items = blocks * p.splits;
  // (threads of a grid: 32 bits)
  return p.items * 64 * p.waves < (int64_t{1} << 32) && batch * q_heads * seq_q <= (int64_t{1} << 31) - 1;
}

bool strides_ok(const int64_t* s) { return s && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0; }

void fill(StreamArgs& a, const Plan& p, const void* q, const int64_t* qs, void* o, const int64_t* os, int64_t batch,
          int64_t q_heads, int64_t kv_heads, int64_t seq_q, int64_t limit, int64_t window, int64_t sinks, float scale,
          void* workspace) {
  a = StreamArgs{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = qs[0], a.q_ss = qs[1], a.q_sh = qs[2];
  a.o = static_cast<uint16_t*>(o);
  a.o_sb = os[0], a.o_ss = os[1], a.o_sh = os[2];
  a.limit = static_cast<int>(limit);
  a.batch = static_cast<int>(batch);
  a.sq = static_cast<int>(seq_q);
  a.hq = static_cast<int>(q_heads);
  a.hkv = static_cast<int>(kv_heads);
  a.group = static_cast<int>(q_heads / kv_heads);
  a.window = static_cast<int>(std::min<int64_t>(window, kMaxSlots));
  a.sinks = static_cast<int>(std::min<int64_t>(sinks, kMaxSlots));
  a.row_tiles = p.row_tiles;
  a.splits = p.splits;
  a.d_group = div_magic(static_cast<uint32_t>(a.group));
  a.d_hkv = div_magic(static_cast<uint32_t>(a.hkv));
  a.d_row_tiles = div_magic(static_cast<uint32_t>(a.row_tiles));
  a.d_splits = div_magic(static_cast<uint32_t>(a.splits));
  a.d_items = div_magic(static_cast<uint32_t>(a.row_tiles) * static_cast<uint32_t>(a.splits));
  a.scale_log2 = scale * kLog2e;
  a.part = static_cast<float*>(workspace);
}

template <int D, int NG, bool kCache, int NW>
void launch_tiles(const StreamArgs& a, dim3 grid, hipStream_t stream) {
  if constexpr (kCache)
    hipLaunchKernelGGL((tile_attn_kernel<D, NG, true, false, NW>), grid, dim3(64 * NW), 0, stream, a);
  else if (a.mask)
    hipLaunchKernelGGL((tile_attn_kernel<D, NG, false, true, NW>), grid, dim3(64 * NW), 0, stream, a);
  else
    hipLaunchKernelGGL((tile_attn_kernel<D, NG, false, false, NW>), grid, dim3(64 * NW), 0, stream, a);
}

template <int D, bool kCache>
hipError_t launch(const StreamArgs& a, const Plan& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.items));
  if (p.rb == kRowsBlock) {
    if (p.waves == 8)
      hipLaunchKernelGGL((rows_attn_kernel<D, kCache, 8>), grid, dim3(64 * 8), 0, stream, a);
    else
      hipLaunchKernelGGL((rows_attn_kernel<D, kCache, 4>), grid, dim3(64 * 4), 0, stream, a);
  } else if (p.rb == 32) {
    launch_tiles<D, 4, kCache, 4>(a, grid, stream);
  } else if (p.rb == 64) {
    if constexpr (kCache)
      launch_tiles<D, 4, true, 8>(a, grid, stream);
    else
      launch_tiles<D, 2, false, 4>(a, grid, stream);
  } else {
    if (p.waves == 8)
      launch_tiles<D, 2, kCache, 8>(a, grid, stream);
    else
      launch_tiles<D, 1, kCache, 4>(a, grid, stream);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  const int per = p.splits <= kMaxSplits / kWaves ? 1 : kWaves;  // waves to a row
  const int64_t out_rows = static_cast<int64_t>(a.batch) * a.hq * a.sq;
  hipLaunchKernelGGL((merge_kernel<D, kCache>), dim3(static_cast<unsigned>((out_rows * per + kWaves - 1) / kWaves)),
                     dim3(64 * kWaves), 0, stream, a, p.rb, per);
  return hipGetLastError();
}

// (scale 0 or below, infinite or NaN is refused)
bool common_ok(const void* q, const int64_t* qs, const void* o, const int64_t* os, float scale) {
  return strides_ok(qs) && strides_ok(os) && scale > 0.f && scale < __builtin_inff() && a16(q) && a16(o);
}

}  // namespace
}  // namespace rldx

using namespace rldx;

extern "C" int64_t rldx_window_attention_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                         int64_t seq_q, int64_t seq_k, int64_t head_dim,
                                                         int64_t window, int64_t sinks) {
  Plan p;
  if (seq_q > seq_k || !plan_of(p, batch, q_heads, kv_heads, seq_q, seq_k, head_dim, window, sinks, false)) return -1;
  return p.workspace(head_dim);
}

extern "C" hipError_t rldx_window_attention_bf16(const void* q, const int64_t* q_strides, const void* k,
                                                 const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                                 void* o, const int64_t* o_strides, int64_t batch, int64_t q_heads,
                                                 int64_t kv_heads, int64_t seq_q, int64_t seq_k, int64_t head_dim,
                                                 int64_t window, int64_t sinks, const float* key_mask,
                                                 int64_t key_mask_batch_stride, float scale, void* workspace,
                                                 int64_t workspace_bytes, hipStream_t stream) {
  Plan p;
  if (seq_q > seq_k || !plan_of(p, batch, q_heads, kv_heads, seq_q, seq_k, head_dim, window, sinks, false) ||
      !common_ok(q, q_strides, o, o_strides, scale) || !strides_ok(k_strides) || !strides_ok(v_strides) || !a16(k) ||
      !a16(v) || reinterpret_cast<uintptr_t>(key_mask) % 4)
    return hipErrorInvalidValue;
  // (a tile's rows are addressed with 32-bit byte offsets)
  if (k_strides[1] < 0 || v_strides[1] < 0 || k_strides[1] > (1 << 24) || v_strides[1] > (1 << 24))
    return hipErrorInvalidValue;
  if (batch == 0 || q_heads == 0 || seq_q == 0) return hipSuccess;
  if (!q || !k || !v || !o) return hipErrorInvalidValue;
  if (p.workspace(head_dim) > 0 && (!workspace || !a16(workspace) || workspace_bytes < p.workspace(head_dim)))
    return hipErrorInvalidValue;
  StreamArgs a;
  fill(a, p, q, q_strides, o, o_strides, batch, q_heads, kv_heads, seq_q, seq_k, window, sinks, scale, workspace);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.k_sb = k_strides[0], a.k_ss = k_strides[1], a.k_sh = k_strides[2];
  a.v_sb = v_strides[0], a.v_ss = v_strides[1], a.v_sh = v_strides[2];
  a.mask = key_mask;
  a.mask_sb = key_mask_batch_stride;
  return head_dim == 128 ? launch<128, false>(a, p, stream) : launch<64, false>(a, p, stream);
}

extern "C" int64_t rldx_kv4_attention_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads,
                                                      int64_t seq_q, int64_t head_dim, int64_t page_tokens,
                                                      int64_t table_pages, int64_t window, int64_t sinks) {
  Plan p;
  if (rldx_kv4_page_bytes(page_tokens, head_dim) < 0 || table_pages < 0 || table_pages > kMaxSlots / page_tokens ||
      !plan_of(p, batch, q_heads, kv_heads, seq_q, table_pages * page_tokens, head_dim, window, sinks, true))
    return -1;
  return p.workspace(head_dim);
}

extern "C" hipError_t rldx_kv4_attention_bf16(const void* q, const int64_t* q_strides, const rldx_kv4_cache_t* cache,
                                              const int32_t* starts, const int32_t* counts, void* o,
                                              const int64_t* o_strides, int64_t batch, int64_t q_heads, int64_t seq_q,
                                              int64_t window, int64_t sinks, float scale, void* workspace,
                                              int64_t workspace_bytes, hipStream_t stream) {
  Plan p;
  if (!kv4_cache_ok(cache) || !common_ok(q, q_strides, o, o_strides, scale) ||
      !plan_of(p, batch, q_heads, cache->kv_heads, seq_q, cache->table_pages * cache->page_tokens, cache->head_dim,
               window, sinks, true))
    return hipErrorInvalidValue;
  if (batch == 0 || q_heads == 0 || seq_q == 0) return hipSuccess;
  if (!q || !o || !starts) return hipErrorInvalidValue;
  if (p.workspace(cache->head_dim) > 0 &&
      (!workspace || !a16(workspace) || workspace_bytes < p.workspace(cache->head_dim)))
    return hipErrorInvalidValue;
  StreamArgs a;
  fill(a, p, q, q_strides, o, o_strides, batch, q_heads, cache->kv_heads, seq_q,
       cache->table_pages * cache->page_tokens, window, sinks, scale, workspace);
  a.cache = static_cast<const uint8_t*>(cache->data);
  a.page_stride = cache->page_stride;
  a.head_stride = cache->head_stride;
  a.num_pages = static_cast<int>(cache->num_pages);
  a.page_shift = __builtin_ctzll(static_cast<unsigned long long>(cache->page_tokens));
  a.table = cache->page_table;
  a.table_sb = cache->page_table_stride;
  a.starts = starts;
  a.counts = counts;
  return cache->head_dim == 128 ? launch<128, true>(a, p, stream) : launch<64, true>(a, p, stream);
}
