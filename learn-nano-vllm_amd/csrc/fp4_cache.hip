// The 4-bit cache as it is written and read back (layout: fp4.h).
//
//   store   keys and values of new tokens, quantised as they are scattered by slot_mapping
//           (what nvk_kv_store is to the 16-bit caches, nanovllm/layers/attention.py:10-40);
//   load    the rows of given slots as 16-bit keys and values.
//
// Both are streams: 2 * 2 D bytes per (token, kv head) on the 16-bit side, 2 * (D/2 + D/16) on the
// other.  A thread owns 8 dimensions (16 bytes) of a row's key and value, D / 8 neighbouring
// lanes a row, and the rows of a workgroup are tokens of ONE head: their codes are neighbours
// in the cache wherever their slots are.
//
// One row per thread: 16384 tokens x 8 heads x 128 of consecutive pages are stored in 19.4 us (4.5 TB/s;
// a copy of 1 GiB reaches 5.1) and read back, just written, in 14.5; 64 tokens in 3.1 and 2.9 us.
// 2, 4 and 8 rows per thread: stored in 18.9 / 20.7 / 23.1 us, and 4096 tokens in 8.0 / 8.7 / 9.6
// against 7.0.  The codes are read with plain loads: non-temporal ones take 5 % less time where the
// codes come from HBM (35000 tokens 40.9 / 43.0 us), 30 % more where they were just written.
// Non-temporal stores of the rows end the read-back sooner and make whoever reads them later: 35000
// tokens 34 us against 42, with a reader behind it 91.3 against 90.2; 8300 tokens 9.5 against 12.3, and
// 28.1 against 26.1.
#include "fp4.h"

namespace {

// Grids: heads, pieces of the tokens, and beyond kGridY pieces more of those along z.  Heads first: the
// workgroups of one piece, which share its rows on the 16-bit side, run side by side, and (8 heads) a
// head stays on one of the 8 XCDs, each with an L2 of its own: 16 tokens' scales are a quarter of a
// line.  Pieces first: 16384 tokens stored and read back 34.1 us, not 31.9; 38176 read back 45.0, not
// 43.9; with four neighbouring pieces to one XCD 32.5 and 46.6.
constexpr int kGridY = 32768;
dim3 heads_first(int heads, int64_t pieces) {
  return dim3(heads, (unsigned)(pieces < kGridY ? pieces : kGridY),
              (unsigned)((pieces + kGridY - 1) / kGridY));
}

struct CacheArgs {
  uint8_t *k_data, *v_data;
  uint16_t *k_scale, *v_scale;
  const int32_t* slots;
  int64_t n_tokens;
  int num_kv_heads, block_size, bs_shift;
  int64_t cache_slots;
};

// Head `h` row of a slot: its index among the cache's rows, and its first scale's.
template <int HD>
__device__ __forceinline__ void locate(const CacheArgs& a, int slot, int h, int64_t& row,
                                       int64_t& scale) {
  const int page = a.bs_shift >= 0 ? slot >> a.bs_shift : slot / a.block_size;
  const int off = slot - page * a.block_size;
  const int64_t head = (int64_t)page * a.num_kv_heads + h;
  row = head * a.block_size + off;
  scale = head * (HD / kFp4Group) * a.block_size + off;
}

// The largest magnitude of the 32 dimensions that four neighbouring lanes hold, as the bits of
// |x| (an infinity, then NaN, are the largest).
__device__ __forceinline__ uint32_t group_top(const nvk_u32x4& w) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  uint32_t t = m[0] > m[1] ? m[0] : m[1];
  uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)t, NVK_DPP_QP_XOR1, 0xF, 0xF, true);
  t = o > t ? o : t;
  o = (uint32_t)__builtin_amdgcn_mov_dpp((int)t, NVK_DPP_QP_XOR2, 0xF, 0xF, true);
  return o > t ? o : t;
}

// Codes of 8 elements and the scale of their group.  x / scale is compared with the borders between
// codes, multiples of scale with at most 14 significant bits, as x has at most 11: unless they are
// equal they differ by 2^-14 and more, and x * (1 / scale), corrected once, is exact where they
// are equal.  So the code is the one that exact arithmetic gives.
template <bool F16>
__device__ __forceinline__ uint32_t quantise(const nvk_u32x4& w, uint16_t& scale) {
  using E = NvkElt<F16>;
  const uint32_t top = group_top(w);
  const bool finite = top < (F16 ? 0x7c00u : 0x7f80u);
  const float q = fminf(E::lo(top) / 6.f, 65504.f);
  const _Float16 h = (_Float16)q;
  const float s = (float)h;
  scale = finite ? __builtin_bit_cast(uint16_t, h) : (uint16_t)0x7e00;
  const float inv = finite && s > 0.f ? 1.f / s : 0.f;
  uint32_t code = 0;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = i & 1 ? E::hi(w[i / 2]) : E::lo(w[i / 2]);
    const float p = x * inv;
    y[i] = finite ? fmaf(fmaf(-p, s, x), inv, p) : 0.f;
  }
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[0], y[1], 1.f, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], 1.f, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[4], y[5], 1.f, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[6], y[7], 1.f, 3);
  return code;
}

template <int HD, bool F16>
__global__ __launch_bounds__(256) void fp4_store_kernel(CacheArgs a, const uint16_t* key,
                                                        int64_t key_stride, const uint16_t* value,
                                                        int64_t value_stride) {
  constexpr int kLanes = HD / 8, kRows = 256 / kLanes;  // lanes of a row, rows of a workgroup
  const int u = threadIdx.x % kLanes;
  const int h = blockIdx.x;
  const int64_t t = ((int64_t)blockIdx.z * kGridY + blockIdx.y) * kRows + threadIdx.x / kLanes;
  if (t >= a.n_tokens) return;  // whole rows: the lanes of a group leave together
  const int64_t col = (int64_t)h * HD + 8 * u;
  const int slot = a.slots[t];  // the rows are loaded whatever it is: they do not wait for it
  const nvk_u32x4 k = __builtin_nontemporal_load(
      reinterpret_cast<const nvk_u32x4*>(key + t * key_stride + col));
  const nvk_u32x4 v = __builtin_nontemporal_load(
      reinterpret_cast<const nvk_u32x4*>(value + t * value_stride + col));
  if (slot < 0 || slot >= a.cache_slots) return;
  int64_t row, srow;
  locate<HD>(a, slot, h, row, srow);
  uint16_t ks, vs;
  const uint32_t kc = quantise<F16>(k, ks), vc = quantise<F16>(v, vs);
  *reinterpret_cast<uint32_t*>(a.k_data + row * (HD / 2) + 4 * fp4_place<HD, true>(u)) = kc;
  *reinterpret_cast<uint32_t*>(a.v_data + row * (HD / 2) + 4 * u) = vc;
  if (u % 4 == 0) {
    a.k_scale[srow + (int64_t)(u / 4) * a.block_size] = ks;
    a.v_scale[srow + (int64_t)(u / 4) * a.block_size] = vs;
  }
}

// 8 values from their codes and their group's scale: the products are exact in f32 and rounded once.
template <bool F16>
__device__ __forceinline__ nvk_u32x4 values(uint32_t code, uint16_t scale) {
  using E = NvkElt<F16>;
  const float s = (float)__builtin_bit_cast(_Float16, scale);
  const auto c = __builtin_bit_cast(nvk_u32x4, fp4_unpack<F16>(code));
  nvk_u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = E::pack2(E::lo(c[i]) * s, E::hi(c[i]) * s);
  return o;
}

template <int HD, bool F16>
__global__ __launch_bounds__(256) void fp4_load_kernel(CacheArgs a, uint16_t* key,
                                                       int64_t key_stride, uint16_t* value,
                                                       int64_t value_stride) {
  constexpr int kLanes = HD / 8, kRows = 256 / kLanes;
  const int u = threadIdx.x % kLanes;
  const int h = blockIdx.x;
  const int64_t t = ((int64_t)blockIdx.z * kGridY + blockIdx.y) * kRows + threadIdx.x / kLanes;
  if (t >= a.n_tokens) return;
  const int slot = a.slots[t];
  nvk_u32x4 k = {0u, 0u, 0u, 0u}, v = k;
  if (slot >= 0 && slot < a.cache_slots) {
    int64_t row, srow;
    locate<HD>(a, slot, h, row, srow);
    srow += (int64_t)(u / 4) * a.block_size;
    const uint32_t kc = *reinterpret_cast<const uint32_t*>(a.k_data + row * (HD / 2) +
                                                           4 * fp4_place<HD, true>(u));
    const uint32_t vc = *reinterpret_cast<const uint32_t*>(a.v_data + row * (HD / 2) + 4 * u);
    k = values<F16>(kc, a.k_scale[srow]);
    v = values<F16>(vc, a.v_scale[srow]);
  }
  const int64_t col = (int64_t)h * HD + 8 * u;
  *reinterpret_cast<nvk_u32x4*>(key + t * key_stride + col) = k;
  *reinterpret_cast<nvk_u32x4*>(value + t * value_stride + col) = v;
}

// Prefix sums of a batch whose sequences all have a.n_query queries, by one workgroup.
__device__ void uniform_prefix(const Fp4Expand& a) {
  __shared__ int s_sum[256];
  const int per = (a.total_batch + 255) / 256, b0 = threadIdx.x * per;
  int local = 0;
  for (int i = 0; i < per; ++i)
    if (b0 + i < a.total_batch) local += a.lens[b0 + i];
  s_sum[threadIdx.x] = local;
  __syncthreads();
  int run = 0;
  for (int t = 0; t < (int)threadIdx.x; ++t) run += s_sum[t];
  for (int i = 0; i < per; ++i) {
    if (b0 + i >= a.total_batch) break;
    a.cu_q_out[b0 + i] = (b0 + i) * a.n_query;
    a.cu_k_out[b0 + i] = run;
    run += a.lens[b0 + i];
    if (b0 + i + 1 == a.total_batch) {
      a.cu_q_out[a.total_batch] = a.total_batch * a.n_query;
      a.cu_k_out[a.total_batch] = run;
    }
  }
}

// Keys and values of each sequence's pages as f16 (see Fp4Expand).  grid = (pairs of heads, 16-token
// pieces of a sequence, sequences); 16 lanes a row.  32 sequences of U{612..1536} tokens and 8 heads,
// 37 MB read and 133 written: 33 to 36 us.  Pieces first 39; in that order all heads of a piece in a
// workgroup 41, one head 48, and other mappings (a quad per row, 4 heads of a token per wave, loads a step
// ahead) 41 to 48.
template <bool F16>
__global__ __launch_bounds__(256) void fp4_expand_kernel(Fp4Expand a) {
  constexpr int HD = 128, HB = 2;
  const int folds = (a.pages_per_seq * (kFp4Page / 16) + kGridY - 1) / kGridY;
  const int s = folds == 1 ? blockIdx.z : blockIdx.z / folds;
  const int piece = (blockIdx.z - s * folds) * kGridY + blockIdx.y, h0 = HB * blockIdx.x;
  if (piece == 0 && h0 == 0) {
    for (int i = threadIdx.x; i < a.pages_per_seq; i += 256)
      a.tables[(int64_t)s * a.pages_per_seq + i] = s * a.pages_per_seq + i;
    if (a.cu_q_out && s == 0) uniform_prefix(a);
  }
  // the page is looked up beside the length, not after it
  const int u = threadIdx.x % 16;
  const int p = piece * 16 + threadIdx.x / 16;
  const int logical = a.bs_shift >= 0 ? p >> a.bs_shift : p / a.block_size;
  int page = a.block_tables[s * a.bt_stride + min(logical, a.max_blocks - 1)];
  int64_t keys = a.lens ? a.lens[a.first + s] : (int64_t)a.cu_k[s + 1] - a.cu_k[s];
  if (keys > (int64_t)a.pages_per_seq * kFp4Page) keys = (int64_t)a.pages_per_seq * kFp4Page;
  if (keys > (int64_t)a.max_blocks * a.block_size) keys = (int64_t)a.max_blocks * a.block_size;
  if (p >= keys) return;  // whole rows
  if (page < 0 || page >= a.num_blocks) page = 0;
  const int off = p - logical * a.block_size;
  const int64_t head0 = (int64_t)page * a.num_kv_heads;
  uint32_t kc[HB], vc[HB];
  uint16_t ks[HB], vs[HB];
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    const int64_t head = head0 + min(h0 + i, a.num_kv_heads - 1);
    const int64_t row = head * a.block_size + off;
    const int64_t srow = head * 4 * a.block_size + off + (int64_t)(u / 4) * a.block_size;
    kc[i] = *reinterpret_cast<const uint32_t*>(a.k_data + row * (HD / 2) +
                                               4 * fp4_place<HD, true>(u));
    vc[i] = *reinterpret_cast<const uint32_t*>(a.v_data + row * (HD / 2) + 4 * u);
    ks[i] = a.k_scale[srow];
    vs[i] = a.v_scale[srow];
  }
  // products of f16 numbers (the codes exact, times 2^-kFp4KeyShift or 1), each rounded once
  auto f16_values = [](uint32_t code, _Float16 s) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    constexpr float kUnit = F16 ? 1.f : 1.f / (1 << kFp4KeyShift);
    const h2 ss = {s, s}, top = {(_Float16)65504.f, (_Float16)65504.f};
    h2 c[4] = {__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, kUnit, 0),
               __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, kUnit, 1),
               __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, kUnit, 2),
               __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(code, kUnit, 3)};
    nvk_u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] *= ss;
      // (min and max drop a NaN: it goes into the keys below)
      if constexpr (F16) c[i] = __builtin_elementwise_max(__builtin_elementwise_min(c[i], top), -top);
      o[i] = __builtin_bit_cast(uint32_t, c[i]);
    }
    return o;
  };
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    const int h = h0 + i;
    if (h >= a.num_kv_heads) continue;  // uniform
    // A value that is not finite would meet the zero probability of a query that does not see
    // it, as NaN.  It becomes 0 here and the row's key NaN, whose score a mask replaces.
    const bool v_lost = (vs[i] & 0x7c00) == 0x7c00;
    const bool lost = v_lost || (ks[i] & 0x7c00) == 0x7c00;
    const bool row_lost = (__builtin_amdgcn_ballot_w64(lost) >> (threadIdx.x & 48) & 0xffffu) != 0;
    nvk_u32x4 k = f16_values(kc[i], __builtin_bit_cast(_Float16, ks[i]));
    const nvk_u32x4 v =
        f16_values(vc[i], v_lost ? (_Float16)0.f : __builtin_bit_cast(_Float16, vs[i]));
    if (row_lost) k = nvk_u32x4{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u};
    const int64_t at =
        (((int64_t)s * a.pages_per_seq * kFp4Page + p) * a.num_kv_heads + h) * HD + 8 * u;
    *reinterpret_cast<nvk_u32x4*>(a.k_pages + at) = k;
    *reinterpret_cast<nvk_u32x4*>(a.v_pages + at) = v;
  }
}

// The checks that store and load share; fills `a`.
int cache_args(CacheArgs& a, const void* rows_k, int64_t key_row_stride, const void* rows_v,
               int64_t value_row_stride, void* k_data, void* k_scale, void* v_data, void* v_scale,
               const int32_t* slots, int64_t n_tokens, int32_t num_kv_heads, int32_t head_dim,
               int32_t block_size, int32_t num_blocks, int32_t dtype) {
  if (n_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks < 0)
    return NVK_EINVAL;
  if (dtype != NVK_DTYPE_BF16 && dtype != NVK_DTYPE_F16) return NVK_EUNSUPPORTED;
  if ((head_dim != 128 && head_dim != 64) || block_size % 16) return NVK_EUNSUPPORTED;
  const int64_t cache_slots = (int64_t)num_blocks * block_size;
  if (num_kv_heads > 65535 || n_tokens > (int64_t)INT32_MAX) return NVK_EINVAL;
  if (n_tokens == 0) return NVK_OK;
  if (!rows_k || !rows_v || !k_data || !k_scale || !v_data || !v_scale || !slots)
    return NVK_EINVAL;
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key_row_stride < row || value_row_stride < row) return NVK_EINVAL;
  if (((uintptr_t)rows_k | (uintptr_t)rows_v | (uintptr_t)k_data | (uintptr_t)v_data |
       (uintptr_t)k_scale | (uintptr_t)v_scale) % 16 ||
      (uintptr_t)slots % 4 || key_row_stride % 8 || value_row_stride % 8)
    return NVK_EALIGN;
  a.k_data = static_cast<uint8_t*>(k_data);
  a.v_data = static_cast<uint8_t*>(v_data);
  a.k_scale = static_cast<uint16_t*>(k_scale);
  a.v_scale = static_cast<uint16_t*>(v_scale);
  a.slots = slots;
  a.n_tokens = n_tokens;
  a.num_kv_heads = num_kv_heads;
  a.block_size = block_size;
  a.bs_shift = nvk_log2_exact(block_size);
  a.cache_slots = cache_slots;
  return NVK_OK;
}

// f(std::integral_constant head size, std::bool_constant f16)
template <typename F>
int by_type(int head_dim, int dtype, F&& f) {
  const bool f16 = dtype == NVK_DTYPE_F16;
  if (head_dim == 128)
    return f16 ? f.template operator()<128, true>() : f.template operator()<128, false>();
  return f16 ? f.template operator()<64, true>() : f.template operator()<64, false>();
}

struct StoreLaunch {
  const CacheArgs& a;
  const uint16_t *k, *v;
  int64_t ks, vs;
  hipStream_t s;
  template <int HD, bool F16>
  int operator()() const {
    constexpr int kRows = 256 / (HD / 8);
    const dim3 grid = heads_first(a.num_kv_heads, (a.n_tokens + kRows - 1) / kRows);
    hipLaunchKernelGGL((fp4_store_kernel<HD, F16>), grid, dim3(256), 0, s, a, k, ks, v, vs);
    return nvk_launch_status();
  }
};

struct LoadLaunch {
  const CacheArgs& a;
  uint16_t *k, *v;
  int64_t ks, vs;
  hipStream_t s;
  template <int HD, bool F16>
  int operator()() const {
    constexpr int kRows = 256 / (HD / 8);
    const dim3 grid = heads_first(a.num_kv_heads, (a.n_tokens + kRows - 1) / kRows);
    hipLaunchKernelGGL((fp4_load_kernel<HD, F16>), grid, dim3(256), 0, s, a, k, ks, v, vs);
    return nvk_launch_status();
  }
};

}  // namespace

int fp4_expand_launch(const Fp4Expand& p, hipStream_t stream) {
  dim3 grid = heads_first((p.num_kv_heads + 1) / 2, (int64_t)p.pages_per_seq * (kFp4Page / 16));
  grid.z *= p.batch;
  if (p.f16)
    hipLaunchKernelGGL(fp4_expand_kernel<true>, grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(fp4_expand_kernel<false>, grid, dim3(256), 0, stream, p);
  return nvk_launch_status();
}

extern "C" int nvk_fp4_store(const void* key, int64_t key_row_stride, const void* value,
                             int64_t value_row_stride, void* k_data, void* k_scale, void* v_data,
                             void* v_scale, const int32_t* slot_mapping, int64_t n_tokens,
                             int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                             int32_t num_blocks, int32_t dtype, void* stream) {
  CacheArgs a;
  const int st = cache_args(a, key, key_row_stride, value, value_row_stride, k_data, k_scale,
                            v_data, v_scale, slot_mapping, n_tokens, num_kv_heads, head_dim,
                            block_size, num_blocks, dtype);
  if (st != NVK_OK || n_tokens == 0) return st;
  return by_type(head_dim, dtype,
                 StoreLaunch{a, static_cast<const uint16_t*>(key),
                             static_cast<const uint16_t*>(value), key_row_stride,
                             value_row_stride, reinterpret_cast<hipStream_t>(stream)});
}

extern "C" int nvk_fp4_load(const void* k_data, const void* k_scale, const void* v_data,
                            const void* v_scale, const int32_t* slot_mapping, int64_t n_tokens,
                            int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                            int32_t num_blocks, void* key, int64_t key_row_stride, void* value,
                            int64_t value_row_stride, int32_t dtype, void* stream) {
  CacheArgs a;
  const int st =
      cache_args(a, key, key_row_stride, value, value_row_stride, const_cast<void*>(k_data),
                 const_cast<void*>(k_scale), const_cast<void*>(v_data), const_cast<void*>(v_scale),
                 slot_mapping, n_tokens, num_kv_heads, head_dim, block_size, num_blocks, dtype);
  if (st != NVK_OK || n_tokens == 0) return st;
  return by_type(head_dim, dtype,
                 LoadLaunch{a, static_cast<uint16_t*>(key), static_cast<uint16_t*>(value),
                            key_row_stride, value_row_stride,
                            reinterpret_cast<hipStream_t>(stream)});
}
