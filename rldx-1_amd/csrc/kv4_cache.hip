// Writing and reading the 4-bit K/V cache (format and layout: kv4_cache.h).
#include <algorithm>

#include "kv4_cache.h"

namespace rldx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Kv4Args {
  uint8_t* cache;
  int64_t page_stride, head_stride;  // bytes
  int num_pages, page_shift;
  const int32_t* table;
  int64_t table_sb;
  int capacity;  // slots of a sequence's row of the table
  const int32_t* starts;
  const int32_t* counts;  // may be null: every row
  int seq, heads, batch;
  // append: sources; read: destinations
  uint16_t *k, *v;
  int64_t k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
};

// Tile of a slot of sequence b in head h, or null (a slot outside the table, a page outside the cache).
__device__ __forceinline__ uint8_t* tile_of(const Kv4Args& a, int b, int64_t slot, int h, int D) {
  if (slot < 0 || slot >= a.capacity) return nullptr;
  const int page = a.table[b * a.table_sb + (slot >> a.page_shift)];
  if (page < 0 || page >= a.num_pages) return nullptr;
  const int in = static_cast<int>(slot) & ((1 << a.page_shift) - 1);
  return a.cache + page * a.page_stride + h * a.head_stride + (in / kv4::kTile) * kv4::tile_bytes(D);
}

// One workgroup per tile of the cache that the rows reach, one thread per 8 dimensions of a row of K and of V; the 4
// threads of a block of 32 share its largest magnitude.  Bound by the stream: 2 x 2 D bytes of a row in, 2 (D/2 + D/32)
// out.  4 x 8192 rows of 8 heads of 128, 170 MB: 37 us, 4.6 TB/s (a copy of that size reaches 4.9).  A thread per row
// piece in the rows' own order (heads next to each other) took 49 us: a line of V codes holds a unit of each of 8 slots,
// which then left through the caches of several XCDs, and every thread divided its way to its row.
template <int D>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Args a) {
  constexpr int TPR = D / 8;  // threads per row
  const int h = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  const int64_t start = a.starts[b];
  const int64_t slot0 = ((start >> 5) + blockIdx.x) * kv4::kTile;
  const int n = a.counts ? min(a.seq, a.counts[b]) : a.seq;
  uint8_t* const t = tile_of(a, b, slot0, h, D);
  if (!t) return;
  const int d0 = static_cast<int>(threadIdx.x) % TPR * 8;
#pragma unroll
  for (int s = static_cast<int>(threadIdx.x) / TPR; s < kv4::kTile; s += 256 / TPR) {
    const int64_t i = slot0 + s - start;
    if (i < 0 || i >= n) continue;  // whole rows: the threads of a block leave together
    const u32x4 kx = *reinterpret_cast<const u32x4*>(a.k + b * a.k_sb + i * a.k_ss + h * a.k_sh + d0);
    const u32x4 vx = *reinterpret_cast<const u32x4*>(a.v + b * a.v_sb + i * a.v_ss + h * a.v_sh + d0);
    uint32_t codes[2];
    uint32_t scale[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const u32x4 x = kv ? vx : kx;
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = x[j];
        m = max(m, max((w << 16) & 0x7fffffffu, w & 0x7fff0000u));
      }
      m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 1)));
      m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 2)));
      const int e = kv4::block_exponent(m);
      // (element_code of two values in one instruction: v_cvt_scalef32_pk_fp4_bf16 divides by the scale, rounds ties to
      // the even code and cuts off at 6)
      const float s2 = __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23);
      const uint32_t w0 = x[0], w1 = x[1], w2 = x[2], w3 = x[3];
      uint32_t c = 0;
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w0), s2, 0);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w1), s2, 1);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w2), s2, 2);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, w3), s2, 3);
      codes[kv] = c;
      scale[kv] = m >= 0x7f800000u ? kv4::kScaleNan : static_cast<uint32_t>(e + 127);
    }
    *reinterpret_cast<uint32_t*>(t + s * (D / 2) + d0 / 2) = codes[0];
    uint8_t* const vt = t + 16 * D;
    if constexpr (D == 128) {
      *reinterpret_cast<uint32_t*>(vt + ((kv4::v_group(s) * 16 + d0 / 8) * 8 + kv4::v_unit(s)) * 4) = codes[1];
    } else {
      uint16_t* const u = reinterpret_cast<uint16_t*>(vt) + (kv4::v_group(s) * 16 + d0 / 4) * 8 + kv4::v_unit(s);
      u[0] = static_cast<uint16_t>(codes[1]);
      u[8] = static_cast<uint16_t>(codes[1] >> 16);
    }
    if (d0 % 32 == 0) {
      t[32 * D + s * (D / 32) + d0 / 32] = static_cast<uint8_t>(scale[0]);
      t[33 * D + (d0 / 32 * 4 + kv4::v_group(s)) * 8 + kv4::v_unit(s)] = static_cast<uint8_t>(scale[1]);
    }
  }
}

__device__ __forceinline__ u32x4 dequant8(uint32_t c, uint32_t scale_byte) {
  const float s = __builtin_bit_cast(float, scale_byte << 23);  // 255: the conversion gives NaN
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}

// The slots starts[b] .. + seq - 1 as bf16 rows; a slot that cannot be read gives NaN.  Tiles and threads as above, for
// the same reason; the rows leave past the L2: the 170 MB take 27 us (33 in the rows' own order, 28 through the L2), twice
// of them 50 (72 through the L2).
template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Args a) {
  constexpr int TPR = D / 8;
  const int h = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  const int64_t start = a.starts[b];
  const int64_t slot0 = ((start >> 5) + blockIdx.x) * kv4::kTile;
  const uint8_t* const t = tile_of(a, b, slot0, h, D);
  const int d0 = static_cast<int>(threadIdx.x) % TPR * 8;
#pragma unroll
  for (int s = static_cast<int>(threadIdx.x) / TPR; s < kv4::kTile; s += 256 / TPR) {
    const int64_t i = slot0 + s - start;
    if (i < 0 || i >= a.seq) continue;
    u32x4 kx, vx;
    if (t) {
      const uint8_t* const vt = t + 16 * D;
      const uint32_t kc = *reinterpret_cast<const uint32_t*>(t + s * (D / 2) + d0 / 2);
      uint32_t vc;
      if constexpr (D == 128) {
        vc = *reinterpret_cast<const uint32_t*>(vt + ((kv4::v_group(s) * 16 + d0 / 8) * 8 + kv4::v_unit(s)) * 4);
      } else {
        const uint16_t* const u =
            reinterpret_cast<const uint16_t*>(vt) + (kv4::v_group(s) * 16 + d0 / 4) * 8 + kv4::v_unit(s);
        vc = u[0] | static_cast<uint32_t>(u[8]) << 16;
      }
      kx = dequant8(kc, t[32 * D + s * (D / 32) + d0 / 32]);
      vx = dequant8(vc, t[33 * D + (d0 / 32 * 4 + kv4::v_group(s)) * 8 + kv4::v_unit(s)]);
    } else {
      kx = vx = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    }
    __builtin_nontemporal_store(kx, reinterpret_cast<u32x4*>(a.k + b * a.k_sb + i * a.k_ss + h * a.k_sh + d0));
    __builtin_nontemporal_store(vx, reinterpret_cast<u32x4*>(a.v + b * a.v_sb + i * a.v_ss + h * a.v_sh + d0));
  }
}

bool a16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Fills `a` for rows k, v [batch, seq, heads, D]; hipErrorInvalidValue, or hipSuccess with *work telling
// whether there is anything to do.
hipError_t kv4_args(Kv4Args& a, const rldx_kv4_cache_t* c, const void* k, const int64_t* ks,
                    const void* v, const int64_t* vs, const int32_t* starts, const int32_t* counts, int64_t batch,
                    int64_t seq, bool* work) {
  *work = false;
  if (!kv4_cache_ok(c) || batch < 0 || seq < 0 || !ks || !vs) return hipErrorInvalidValue;
  if (batch == 0 || seq == 0 || c->kv_heads == 0) return hipSuccess;
  if (!k || !v || !starts || !a16(k) || !a16(v)) return hipErrorInvalidValue;
  for (int i = 0; i < 3; ++i)
    if (ks[i] % 8 || vs[i] % 8) return hipErrorInvalidValue;
  if (seq > (int64_t{1} << 28) || batch > 65535) return hipErrorInvalidValue;
  a.cache = static_cast<uint8_t*>(c->data);
  a.page_stride = c->page_stride;
  a.head_stride = c->head_stride;
  a.num_pages = static_cast<int>(c->num_pages);
  a.page_shift = __builtin_ctzll(static_cast<unsigned long long>(c->page_tokens));
  a.table = c->page_table;
  a.table_sb = c->page_table_stride;
  a.capacity = static_cast<int>(c->table_pages * c->page_tokens);
  a.starts = starts;
  a.counts = counts;
  a.seq = static_cast<int>(seq);
  a.heads = static_cast<int>(c->kv_heads);
  a.batch = static_cast<int>(batch);
  a.k = static_cast<uint16_t*>(const_cast<void*>(k));
  a.v = static_cast<uint16_t*>(const_cast<void*>(v));
  a.k_sb = ks[0], a.k_ss = ks[1], a.k_sh = ks[2];
  a.v_sb = vs[0], a.v_ss = vs[1], a.v_sh = vs[2];
  *work = true;
  return hipSuccess;
}

// tiles that seq rows may reach, from wherever they start
dim3 tile_grid(const Kv4Args& a) {
  return dim3(static_cast<unsigned>((a.seq + 2 * kv4::kTile - 2) / kv4::kTile), static_cast<unsigned>(a.heads),
              static_cast<unsigned>(a.batch));
}

}  // namespace

bool kv4_cache_ok(const rldx_kv4_cache_t* c) {
  if (!c || (c->head_dim != 64 && c->head_dim != 128)) return false;
  if (c->num_pages < 0 || c->num_pages > (int64_t{1} << 31) - 1 || c->kv_heads < 0 || c->kv_heads > 65535) return false;
  if (c->page_tokens < 32 || c->page_tokens > (1 << 20) || (c->page_tokens & (c->page_tokens - 1))) return false;
  if (c->table_pages < 0 || c->table_pages * c->page_tokens > (int64_t{1} << 30)) return false;
  if (c->page_stride % 16 || c->head_stride % 16) return false;
  if (!a16(c->data) || (c->num_pages > 0 && c->kv_heads > 0 && !c->data)) return false;
  if (c->table_pages > 0 && !c->page_table) return false;
  const int64_t bytes = rldx_kv4_page_bytes(c->page_tokens, c->head_dim);
  if (c->kv_heads > 1 && c->head_stride < bytes) return false;
  return c->num_pages <= 1 || c->page_stride >= bytes;
}

}  // namespace rldx

using namespace rldx;

extern "C" int64_t rldx_kv4_page_bytes(int64_t page_tokens, int64_t head_dim) {
  if (page_tokens < 32 || page_tokens > (1 << 20) || (page_tokens & (page_tokens - 1)) ||
      (head_dim != 64 && head_dim != 128))
    return -1;
  return page_tokens / kv4::kTile * kv4::tile_bytes(static_cast<int>(head_dim));
}

extern "C" int rldx_host_kv4_encode_bf16(const void* x, void* codes, void* scales, int64_t blocks) {
  if (blocks < 0 || (blocks > 0 && (!x || !codes || !scales))) return 1;
  const uint16_t* const src = static_cast<const uint16_t*>(x);
  for (int64_t i = 0; i < blocks; ++i) {
    uint32_t m = 0;
    for (int j = 0; j < 32; ++j) m = std::max(m, static_cast<uint32_t>(src[i * 32 + j] & 0x7fff) << 16);
    const int e = kv4::block_exponent(m);
    for (int j = 0; j < 16; ++j)
      static_cast<uint8_t*>(codes)[i * 16 + j] =
          static_cast<uint8_t>(kv4::element_code(bf16_bits_to_f32(src[i * 32 + 2 * j]), e) |
                               kv4::element_code(bf16_bits_to_f32(src[i * 32 + 2 * j + 1]), e) << 4);
    static_cast<uint8_t*>(scales)[i] = static_cast<uint8_t>(m >= 0x7f800000u ? kv4::kScaleNan : e + 127);
  }
  return 0;
}

extern "C" hipError_t rldx_kv4_append_bf16(const rldx_kv4_cache_t* cache, const void* k, const int64_t* k_strides,
                                           const void* v, const int64_t* v_strides, const int32_t* starts,
                                           const int32_t* counts, int64_t batch, int64_t seq, hipStream_t stream) {
  Kv4Args a;
  bool work;
  const hipError_t e = kv4_args(a, cache, k, k_strides, v, v_strides, starts, counts, batch, seq, &work);
  if (e != hipSuccess || !work) return e;
  if (cache->head_dim == 128)
    hipLaunchKernelGGL(kv4_append_kernel<128>, tile_grid(a), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(kv4_append_kernel<64>, tile_grid(a), dim3(256), 0, stream, a);
  return hipGetLastError();
}

extern "C" hipError_t rldx_kv4_read_bf16(const rldx_kv4_cache_t* cache, const int32_t* starts, void* k,
                                         const int64_t* k_strides, void* v, const int64_t* v_strides, int64_t batch,
                                         int64_t seq, hipStream_t stream) {
  Kv4Args a;
  bool work;
  const hipError_t e = kv4_args(a, cache, k, k_strides, v, v_strides, starts, nullptr, batch, seq, &work);
  if (e != hipSuccess || !work) return e;
  if (cache->head_dim == 128)
    hipLaunchKernelGGL(kv4_read_kernel<128>, tile_grid(a), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(kv4_read_kernel<64>, tile_grid(a), dim3(256), 0, stream, a);
  return hipGetLastError();
}
