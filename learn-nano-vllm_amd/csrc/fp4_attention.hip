// Attention over the 4-bit cache (layout: fp4.h): the queries are the last ones of their sequence's
// keys, one per sequence (a decode step) or several (verification, a chunk of a prompt).
//
//   s_j = scale * sum_g ks[j, g] * (q_g . kc[j, g])      over the 32-dimension groups g
//   o   = sum_j p_j vs[j, g] vc[j, g] / sum_j p_j        p = softmax over the visible keys
//
// The codes kc, vc are exact in bf16 and f16, so they are what the matrix instructions multiply, and
// the scales are applied to the products: to the f32 sums of a key's groups (S), and to
// the probabilities (P.V), which become one operand per group.
//   * A wave owns a tile of 16 or 32 rows (query token x query head of a kv head) and streams their
//     keys in chunks of 64; the chunks of all (sequence, kv head, tile) groups are cut into equal
//     contiguous ranges, one per wave.  The waves of a workgroup join a group that is cut between
//     them in LDS; one cut between workgroups leaves (O, m, l) records that a second kernel merges.
//     (Records of every wave: 192 x U{256..4096} keys, 16/2 heads, 34.1 us and not 31.6, 8 x 16 queries
//     over 2000 27.1 and not 19.1.)  Short groups get a workgroup of 4 or 8 waves each.
//   * S^T = K Q^T on v_mfma_f32_16x16x32: operand row m = 4 a + i of key block b is key
//     16 a + 4 b + i of the chunk, so lane (g, r) ends up with the scores of keys 16 g .. +15 of
//     row r in order: the order in which ds_read_b64_tr_b4 hands it the values of a dimension.
//   * O^T = V^T P^T likewise, V^T read transposed from LDS by ds_read_b64_tr_b4.
//   * The probabilities times vs are rounded to f16 for both types of model: 2^-11 relative (bf16: 2^-8),
//     and p <= 1, so that nothing overflows.  Below 2^-14 the step is 2^-24, no coarser than that of
//     the scales themselves.
//   * A chunk's keys go to registers, its values and scales to LDS (DMA).  The next chunk's keys are
//     loaded once the scores have used these, its values and scales after P.V: there is always
//     something in flight, and a second buffer for what goes to LDS gained nothing (64 x
//     U{100..2048}, 16/8 heads: 23.1 us per call with two, 22.3 with one).
// What bounds it.  Ranges, 64 x U{100..2048} keys, 16/8 heads (86 MB of codes and scales), 22 us: 4 us until the
// first chunk has come (prefix, position, page, data: four dependent round trips), 11 to 12 us of
// stream at 5.7 to 6.4 TB/s, 4 us for the merging kernel and its launch.  Without the 128 conversions
// of a chunk it is 1 % shorter, so it is not the arithmetic.  192 x U{256..4096}, 16/16 heads (922
// MB): 154 us, 6.0 TB/s.
#include <type_traits>

#include "fp4.h"

namespace {

constexpr int kR = 16;                   // columns of an MFMA: rows (query x head) of a tile, or half of one
constexpr int kCK = 64;                  // keys of a chunk
constexpr int kWavesPerWG = 4;
constexpr int kMaxWGs = 512;             // two workgroups per CU
constexpr int kMaxBatch = 2048;

typedef __attribute__((address_space(4))) const int32_t const_i32;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef NvkElt<true>::vec8 vec8h;

struct AttnArgs {
  const uint16_t* q;
  int64_t q_stride_tok, q_stride_head, total_q;
  const uint8_t *k_data, *v_data;
  const uint16_t *k_scale, *v_scale;
  const int32_t* cu_q;   // null: n_query queries per sequence, keys[s] its context length
  const int32_t* keys;   // cu_seqlens_k, or context lengths
  const int32_t* block_tables;
  int64_t bt_stride;
  int batch, n_query, tile_rows, max_tiles, cap, block_size, num_blocks;
  int bs_shift;          // log2 of block_size, or -1
  int num_kv_heads, G;
  uint32_t g_inverse;    // ceil(2^32 / G): rows (below 2^27) / G as a high product (G > 1)
  float scale_log2;
  uint16_t* out;
  int64_t out_stride_tok, out_stride_head;
  int32_t* desc;  // [batch][Hkv][max_tiles] x 2: first and last workgroup of the group, -1 if empty
  float* rec;     // [workgroups][2][rec_rows][HD + 4]: O, m, l
  int rec_rows, n_waves, wave_shift;  // n_waves = 2^wave_shift
  int round;      // WHOLE: sequences whose groups fill the CUs once, 0: in their own order
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Queries, their first row and the keys of sequence s (cu_q beyond what q holds is not followed).
struct Seq {
  int row0, queries, raw_keys, keys;
};
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int s) {
  Seq x;
  if (a.cu_q) {
    const const_i32* cq = (const_i32*)a.cu_q;
    const const_i32* ck = (const_i32*)a.keys;
    x.row0 = cq[s];
    x.queries = cq[s + 1] - x.row0;
    x.raw_keys = ck[s + 1] - ck[s];
    if (x.queries > a.n_query) x.queries = a.n_query;
    if (x.row0 < 0 || x.queries < 0 || (int64_t)x.row0 + x.queries > a.total_q) x.queries = 0;
  } else {
    x.row0 = s * a.n_query;
    x.queries = a.n_query;
    x.raw_keys = ((const_i32*)a.keys)[s];
  }
  x.keys = x.raw_keys < 0 ? 0 : x.raw_keys;
  if (x.keys > a.cap) x.keys = a.cap;
  return x;
}
__device__ __forceinline__ int tiles_of(const AttnArgs& a, const Seq& x) {
  return (x.queries * a.G + a.tile_rows - 1) / a.tile_rows;
}
__device__ __forceinline__ int chunks_of(const Seq& x) { return (x.keys + kCK - 1) / kCK; }
__device__ __forceinline__ int seq_units(const AttnArgs& a, int s) {
  const Seq x = seq_of(a, s);
  return tiles_of(a, x) * chunks_of(x);
}

// Exclusive prefix of the sequences' (tile, chunk) pairs into s_cs[0..B]; returns the total.
__device__ int unit_prefix(const AttnArgs& a, int* s_cs, int* s_wsum) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int B = a.batch;
  if (B <= 64) {  // every wave makes the same one for itself: no barrier
    const int n = lane < B ? seq_units(a, lane) : 0;
    const int x = nvk_wave_scan_add(n);
    if (lane < B) s_cs[lane + 1] = x;
    if (lane == 0) s_cs[0] = 0;
    return __builtin_amdgcn_readlane(x, 63);
  }
  const int per = (B + 255) / 256;
  const int b0 = tid * per;
  int local = 0;
  for (int i = 0; i < per; ++i)
    if (b0 + i < B) local += seq_units(a, b0 + i);
  const int x = nvk_wave_scan_add(local);
  if (lane == 63) s_wsum[wave] = x;
  __syncthreads();
  int run = x - local;
  for (int w = 0; w < wave; ++w) run += s_wsum[w];
  for (int i = 0; i < per; ++i) {
    if (b0 + i < B) {
      s_cs[b0 + i] = run;
      run += seq_units(a, b0 + i);
    }
  }
  const int total = s_wsum[0] + s_wsum[1] + s_wsum[2] + s_wsum[3];
  if (tid == 0) s_cs[B] = total;
  __syncthreads();
  return total;
}

// T chunks over n_waves waves, a power of two: wave w takes [w T / n, (w + 1) T / n), so that the
// waves with one chunk more are spread over the CUs.  Fewer chunks than waves: one each.
struct Split {
  int T, P, shift;
  __device__ __forceinline__ int begin(int w) const {
    return P == T ? w : (int)((int64_t)w * T >> shift);
  }
  __device__ __forceinline__ int owner(int c) const {  // of chunk c; exact: below 2^43, and 53 bits
    return P == T ? c : (int)(((double)((int64_t)(c + 1) << shift) - 1.0) / (double)T);
  }
};

// WHOLE, more groups than CUs: the sequence of place y, such that a CU's groups add up to much the same.
// Places go to the CUs in rounds: by falling length in the first, third, ... round, by rising
// length in those between.  (Every group's result is the same in any order.)  In their own order /
// dealt out: 64 x U{100..2048}, 16/8 heads, 22.7 / 19.5 us, 100 x U{100..1500}, 16/4 heads, 17.9 / 14.9,
// 64 x 6 queries over U{100..1024} 17.9 / 16.1; contexts of one length 29.6 / 30.5 (64 x 2048): it takes
// 1 us, which up to 512 keys is not regained (64 x U{16..256} 7.2 / 8.4).
constexpr int kBalanced = 128;  // sequences, two per lane
template <int W>
__device__ int balanced_place(const AttnArgs& a, int y, int lane, int wave, int (*s_count)[kBalanced]) {
  const int round = y / a.round, p = y - round * a.round;
  const int in_round = min(a.round, a.batch - round * a.round);
  const int rank = round * a.round + (round & 1 ? in_round - 1 - p : p);
  int key[2];  // chunks, then the lower number first: no two alike
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int s = lane + 64 * i;
    key[i] = -1;
    if (s < a.batch) {
      const Seq x = seq_of(a, s);
      key[i] = (x.queries > 0 ? min(chunks_of(x), 1 << 20) : 0) * kBalanced + kBalanced - 1 - s;
    }
  }
  int longer[2] = {0, 0};  // of this wave's share of the sequences
  constexpr int kShare = kBalanced / W;
#pragma unroll
  for (int j = 0; j < kShare; ++j) {
    const int c = wave * kShare + j;
    const int k = __builtin_amdgcn_readlane(c < 64 ? key[0] : key[1], c & 63);
    longer[0] += k > key[0];
    longer[1] += k > key[1];
  }
  s_count[wave][lane] = longer[0];
  s_count[wave][lane + 64] = longer[1];
  __syncthreads();
  int all[2] = {0, 0};
#pragma unroll
  for (int v = 0; v < W; ++v) {
    all[0] += s_count[v][lane];
    all[1] += s_count[v][lane + 64];
  }
  const uint64_t m = __builtin_amdgcn_ballot_w64(lane < a.batch && all[0] == rank);
  if (m) return __builtin_ctzll(m);
  return 64 + __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane + 64 < a.batch && all[1] == rank));
}

// 16 bytes per lane straight into LDS: lane l writes [dst + 16 l, +16).  From base + the lane's
// offset, or from the lane's own address.
__device__ __forceinline__ void lds_load(const void* base, uint32_t offset, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1 nt"
               :: "v"(offset), "s"(base), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void lds_load(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off nt"
               :: "v"(src), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// The wave's LDS reads are done: their buffer may be refilled.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ float sum_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float max_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// (p0, p1) times a pair of f16 scales, each product rounded once to f16: v_fma_mixlo / mixhi_f16,
// which take the scales as they are.  (The empty asm keeps the two roundings apart: a pair of them
// becomes two conversions of the scales, two f32 products and one conversion.)
__device__ __forceinline__ uint32_t times_scales(float p0, float p1, uint32_t scales) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 s = __builtin_bit_cast(h2, scales);
  _Float16 lo = (_Float16)fmaf(p0, (float)s[0], 0.f);
  asm("" : "+v"(lo));
  const h2 d = {lo, (_Float16)fmaf(p1, (float)s[1], 0.f)};
  return __builtin_bit_cast(uint32_t, d);
}

template <int HD>
struct KeyVec;
template <>
struct KeyVec<128> {
  typedef nvk_u32x4 type;
};
template <>
struct KeyVec<64> {
  typedef nvk_u32x2 type;
};

// ONEPAGE: pages of a multiple of 64 keys, so that a chunk lies in one; else of a multiple of 16.
// NC: columns of the 16 that a row takes, for steps of at most 16 / NC rows per kv head (NC = 4: the
// decode of up to 4 heads of 128).  Column (row, c) holds the query in the dimensions of NG / NC of
// the NG = D / 32 groups and zeros elsewhere, so the MFMAs of other columns' groups add nothing to it.
// A score is then NG / NC products with scales in each of NC lanes, which add up, instead of NG in
// one; and a lane needs P vs for its own groups only, whose dimensions alone are kept of its output.
// NT: 16-row blocks of a tile.  Two share what the wave loads and converts (see wide_tiles).
// W waves per workgroup.  WHOLE: a workgroup owns one group (grid = kv heads, sequences, tiles), its
// waves an equal part of the chunks each; they join their states in LDS, and nothing is left to a
// second kernel (see whole_waves).  Waves per SIMD: as many as the registers allow.
template <int HD, bool F16, bool ONEPAGE, int NC, int NT = 1, int W = kWavesPerWG,
          bool WHOLE = false>
__global__ __launch_bounds__(64 * W, WHOLE ? (NC >= 4 || HD == 64 ? 4 : NC == 2 && W == 4 ? 3 : 2)
                                           : 2) void fp4_attention_kernel(AttnArgs a) {
  using E = NvkElt<F16>;
  typedef typename E::vec8 vec8;
  typedef typename KeyVec<HD>::type kvec;
  constexpr int NG = HD / kFp4Group;       // scale groups = MFMA k-steps of S
  constexpr int RB = HD / 2;               // bytes of a row of codes
  constexpr int kVBytes = kCK * RB;        // a chunk's values in LDS
  constexpr int kBuf = kVBytes + 1024;     // and its scales (D = 64 uses half of the 1024)
  constexpr int kBlk = ONEPAGE ? 1 : 4;    // pages looked up per chunk
  constexpr int kRec = HD + 4;
  constexpr int NS = NG / NC;              // groups of a column
  constexpr int kState = WHOLE ? kR / NC * kRec * (int)sizeof(float) : 0;  // of a wave's rows, at the end
  __shared__ __attribute__((aligned(1024))) uint8_t lds[W * (kState > kBuf ? kState : kBuf)];
  __shared__ int s_cs[WHOLE ? 1 : kMaxBatch + 1];
  __shared__ int s_wsum[kWavesPerWG];
  // !WHOLE: what waves 1 .. W - 1 hold of a group that began before them: O, (m, l), whether it ended there
  constexpr int kFollow = WHOLE ? 1 : W - 1;
  __shared__ nvk_f32x4 s_o[kFollow][WHOLE ? 1 : NT * 2 * NS][64];
  __shared__ float2 s_ml[kFollow][NT][64];
  __shared__ int s_ended[kFollow];
  __shared__ int s_count[WHOLE ? W : 1][kBalanced];
  const int tid = threadIdx.x, lane = tid & 63;
  const int r = lane & 15, g = lane >> 4;
  const int Hkv = a.num_kv_heads;

  const int wave = uniform(tid >> 6);
  int T = 0, w = 0, c0, c1;
  // position: sequence s, kv head, tile, chunk k of n
  int s, n, tiles, kvh, tile, k;
  Seq sq;
  if constexpr (WHOLE) {
    kvh = blockIdx.x;
    s = blockIdx.y;
    if (a.round) s = uniform(balanced_place<W>(a, s, lane, wave, s_count));
    tile = blockIdx.z;
    sq = seq_of(a, s);
    n = uniform(chunks_of(sq));
    tiles = 1;
    if (sq.queries * a.G <= tile * kR) return;
    c0 = n * wave / W;
    c1 = n * (wave + 1) / W;
    k = c0;
  } else {
    const int S = unit_prefix(a, s_cs, s_wsum);
    if (blockIdx.x == 0) {  // groups that no wave visits
      const int per = Hkv * a.max_tiles;
      for (int e = tid; e < a.batch * per; e += 256) {
        const int b = e / per;
        if (s_cs[b + 1] == s_cs[b])
          *reinterpret_cast<int2*>(a.desc + 2 * (int64_t)e) = make_int2(-1, -1);
      }
    }
    T = uniform(Hkv * S);
    w = blockIdx.x * W + wave;
  }
  const Split sp{T, T < a.n_waves ? T : a.n_waves, a.wave_shift};
  if constexpr (!WHOLE) {
    if (w >= sp.P) {  // no chunk
      __syncthreads();  // the join's
      return;
    }
    c0 = sp.begin(w);
    c1 = sp.begin(w + 1);
    s = nvk_last_le(s_cs, a.batch, Hkv, c0, lane);
    sq = seq_of(a, s);
    n = uniform(chunks_of(sq));
    tiles = uniform(tiles_of(a, sq));
    const int rr = c0 - Hkv * uniform(s_cs[s]);
    const int unit = uniform(rr / n);
    k = uniform(rr - unit * n);
    kvh = tiles == 1 ? unit : uniform(unit / tiles);
    tile = uniform(unit - kvh * tiles);
  }
  bool started_here = k == 0;

  const uint32_t buf = (uint32_t)uniform((int)(uint32_t)(size_t)(lds_ptr)(lds + wave * kBuf));
  // ds_read_b64_tr_b4: the 16 lanes of group g read 8 bytes (16 dimensions) of keys 16 g .. +15;
  // 16-byte chunks of a row are XOR-swizzled by its number so that they spread over the banks.
  const int sw = HD == 128 ? (r >> 2) & 3 : (r >> 3) & 1;
  const uint32_t tr_row = (uint32_t)((16 * g + r) * RB);
  // DMA source of load j, lane l: bytes 16 (l % kCh) ^ swizzle of row (1024 / RB) j + l / kCh
  constexpr int kCh = RB / 16, kRowsPerLoad = 1024 / RB;
  const int vrow = lane / kCh;
  const int vsw = HD == 128 ? (vrow >> 2) & 3 : (vrow >> 3) & 1;
  const int vbyte = 16 * ((lane % kCh) ^ vsw);
  // scale DMA: tensor, group and 8 keys of this lane (D = 64: both halves of the wave the same)
  const int sl = HD == 128 ? lane : lane & 31;
  const bool s_is_v = sl >= 32 * NG / 4;
  const int s_grp = (sl >> 3) & (NG - 1), s_key = 8 * (sl & 7);
  const char* s_base = reinterpret_cast<const char*>(s_is_v ? a.v_scale : a.k_scale) +
                       2 * (s_grp * a.block_size + (ONEPAGE ? s_key : s_key & 15));
  const uint32_t k_off = (uint32_t)((ONEPAGE ? 16 * (r >> 2) : 0) + (r & 3)) * RB + g * (RB / 4);
  const uint32_t v_off = (uint32_t)vrow * RB + vbyte;
  const uint32_t head_bytes = (uint32_t)a.block_size * RB;        // a (page, head)'s codes
  const uint64_t page_bytes = (uint64_t)head_bytes * Hkv;

  // Byte offsets of a chunk's (16-key blocks') first row of codes, and of the same row's scales.
  struct Where {
    uint64_t row[kBlk], scale[kBlk];
    int in_page;  // ONEPAGE: the chunk's first key in its page
  };
  auto locate = [&](int keys, int ss, int hh, int kk) {
    Where p;
    const const_i32* bt = (const_i32*)(a.block_tables + (int64_t)ss * a.bt_stride);
    // the blocks' pages and places first, so that the loads of the page ids go out together
    const int key0 = kk * kCK;
    int logical = a.bs_shift >= 0 ? key0 >> a.bs_shift : key0 / a.block_size;
    int off = key0 - logical * a.block_size;
    int page[kBlk], offs[kBlk];
    p.in_page = off;
    page[0] = bt[logical];
    offs[0] = off;
#pragma unroll
    for (int b = 1; b < kBlk; ++b) {  // a block past the keys: the last one, nothing of it counts
      const bool more = key0 + 16 * b < keys, next = off + 16 == a.block_size;
      logical += more && next;
      off = !more ? off : next ? 0 : off + 16;
      page[b] = bt[logical];
      offs[b] = off;
    }
#pragma unroll
    for (int b = 0; b < kBlk; ++b) {
      const int pg = page[b] < 0 || page[b] >= a.num_blocks ? 0 : page[b];
      const uint64_t head = (uint64_t)(uint32_t)pg * page_bytes + (uint64_t)(uint32_t)hh * head_bytes;
      p.row[b] = head + (uint32_t)offs[b] * RB;
      p.scale[b] = (head >> 3) + (uint32_t)offs[b] * 2;  // 2 bytes of scale per 16 of codes
    }
    return p;
  };
  // The next chunk of the same sequence and head: mostly further down its page.
  auto locate_next = [&](Where p, int keys, int ss, int hh, int kk) {
    if (ONEPAGE && p.in_page + kCK < a.block_size) {
      p.row[0] += kCK * RB;
      p.scale[0] += kCK * 2;
      p.in_page += kCK;
      return p;
    }
    return locate(keys, ss, hh, kk);
  };
  // v[i] of a lane's block i.  (All four read first: a choice between their addresses would put them in
  // scratch memory.)
  auto pick = [](const uint64_t (&v)[kBlk], int i) {
    if constexpr (kBlk == 1) {
      return v[0];
    } else {
      const uint64_t v0 = v[0], v1 = v[1], v2 = v[2], v3 = v[3];
      const uint64_t lo = i & 1 ? v1 : v0, hi = i & 1 ? v3 : v2;
      return i & 2 ? hi : lo;
    }
  };
  auto issue_keys = [&](const Where& p, kvec (&kraw)[4]) {
    const uint8_t* kp = a.k_data + (kBlk == 1 ? p.row[0] : pick(p.row, r >> 2)) + k_off;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      kraw[b] = __builtin_nontemporal_load(reinterpret_cast<const kvec*>(kp + 4 * b * RB));
  };
  auto issue_rest = [&](const Where& p) {
    lds_load(s_base + (kBlk == 1 ? p.scale[0] : pick(p.scale, s_key >> 4)), buf + kVBytes);
#pragma unroll
    for (int j = 0; j < kVBytes / 1024; ++j) {
      if constexpr (kBlk == 1) {
        lds_load(a.v_data + p.row[0], v_off + 1024u * j, buf + 1024 * j);
      } else {
        const int row = kRowsPerLoad * j + vrow;  // of the chunk
        lds_load(a.v_data + pick(p.row, row >> 4) + ((row & 15) * RB + vbyte), buf + 1024 * j);
      }
    }
  };

  // per-group state
  vec8 qf[NT][NG];
  nvk_f32x4 acc[NT][HD / 16];
  float m_run[NT], l_part[NT][2];
  int tok[NT], head[NT], row_limit[NT], full_limit = 0;
  bool row_valid[NT];
  const int row = r / NC, g0 = r % NC * NS;  // this column's row, and the first of its groups
  auto start_group = [&]() {
    const int diag = sq.raw_keys - sq.queries, rr0 = tile * kR * NT;
    full_limit = uniform(min(sq.keys - 1, diag + rr0 / a.G));            // visible to every row
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int rr = rr0 + kR * t + row;
      tok[t] = a.G == 1 ? rr : (int)__umulhi((uint32_t)rr, a.g_inverse);
      head[t] = kvh * a.G + rr - tok[t] * a.G;
      row_valid[t] = tok[t] < sq.queries;
      row_limit[t] = row_valid[t] ? min(sq.keys - 1, diag + tok[t]) : -1;  // last visible key
      const uint16_t* qp = a.q + (int64_t)(sq.row0 + tok[t]) * a.q_stride_tok +
                           (int64_t)head[t] * a.q_stride_head + 8 * g;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        nvk_u32x4 v = {0u, 0u, 0u, 0u};
        if (row_valid[t] && (NC == 1 || i / NS * NS == g0))
          v = *reinterpret_cast<const nvk_u32x4*>(qp + 32 * i);
        qf[t][i] = __builtin_bit_cast(vec8, v);
      }
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) acc[t][d] = nvk_f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[t] = -INFINITY;
      l_part[t][0] = l_part[t][1] = 0.f;
    }
  };

  // the d blocks that are kept of this lane's column, those of its groups; d0: dimension of o[0][0]
  constexpr int kKeep = 2 * NS;
  const int d0 = 32 * g0 + 4 * g;
  auto kept = [&](nvk_f32x4 (&o)[kKeep], int t) {
#pragma unroll
    for (int j = 0; j < kKeep; ++j) {
      o[j] = acc[t][j];
#pragma unroll
      for (int i = 1; i < NC; ++i)
        if (g0 == i * NS) o[j] = acc[t][i * kKeep + j];
    }
  };

  auto put_rows = [&](const nvk_f32x4 (&o)[kKeep], float l, int t) {
    if (!row_valid[t]) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* op = a.out + (int64_t)(sq.row0 + tok[t]) * a.out_stride_tok +
                   (int64_t)head[t] * a.out_stride_head + d0;
#pragma unroll
    for (int j = 0; j < kKeep; ++j) {
      nvk_u32x2 wv;
      wv.x = E::pack2(o[j][0] * inv, o[j][1] * inv);
      wv.y = E::pack2(o[j][2] * inv, o[j][3] * inv);
      *reinterpret_cast<nvk_u32x2*>(op + 16 * j) = wv;
    }
  };
  // The workgroup's record of the group that goes on behind it (0), or began before it (1).
  auto put_record = [&](const nvk_f32x4 (&o)[kKeep], float m, float l, int t) {
    if (!row_valid[t]) return;  // the merge reads the valid rows only
    float* rec = a.rec + ((int64_t)(blockIdx.x * 2 + (started_here ? 0 : 1)) * a.rec_rows + kR * t +
                          row) * kRec;
#pragma unroll
    for (int j = 0; j < kKeep; ++j) *reinterpret_cast<nvk_f32x4*>(rec + d0 + 16 * j) = o[j];
    if (g == 0 && g0 == 0) {
      rec[HD] = m;
      rec[HD + 1] = l;
    }
  };

  kvec kraw[4];
  Where at;
  bool cut = false;  // the range ends inside a group
  if (!WHOLE || c0 < c1) {
    at = locate(sq.keys, s, kvh, k);
    issue_keys(at, kraw);
    issue_rest(at);
  }
  start_group();
  // the next group
  int ns = s, nkvh = kvh, ntile = tile, nn = n, ntiles = tiles;
  Seq nsq = sq;

  for (int c = c0; !WHOLE || c < c1; ++c) {
    // ---- the next chunk: its keys go out once this one's are used, its values and scales at the end
    const bool last = c + 1 == c1;
    const bool group_end = !WHOLE && k == n - 1;
    if (!last) {
      if (!group_end) {
        at = locate_next(at, sq.keys, s, kvh, k + 1);
      } else {
        if (++ntile == tiles) {
          ntile = 0;
          if (++nkvh == Hkv) {
            nkvh = 0;
            int b = s + 1;
            while (s_cs[b + 1] == s_cs[b]) ++b;  // a next chunk exists
            ns = uniform(b);
            nsq = seq_of(a, ns);
            nn = uniform(chunks_of(nsq));
            ntiles = uniform(tiles_of(a, nsq));
          }
        }
        at = locate(nsq.keys, ns, nkvh, 0);
      }
    }
    wait_loads();

    // ---- scores of keys 16 g + 4 b + i, row r
    const int kbase = k * kCK;
    nvk_f32x4 sc[NT][4];
    auto scales = [&](int tensor, int i) {  // of this lane's 16 keys
      return (const __attribute__((address_space(3))) nvk_f16x8*)(size_t)(
          buf + kVBytes + (uint32_t)(128 * (NG * tensor + i) + 32 * g));
    };
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const auto* kp = scales(0, g0 + j);
      const nvk_f16x8 ks[2] = {kp[0], kp[1]};
      nvk_f32x4 x[NT][4] = {};
#pragma unroll
      for (int i = j; i < NG; i += NS)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const vec8 kf = fp4_unpack<F16>(kraw[b][i]);
#pragma unroll
          for (int t = 0; t < NT; ++t) x[t][b] = E::mfma16x16x32(kf, qf[t][i], x[t][b]);
        }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sc[t][b][e] = fmaf(x[t][b][e], (float)ks[b >> 1][4 * (b & 1) + e], j ? sc[t][b][e] : 0.f);
      if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);  // a group's operands at a time
    }
    static_assert(NC == 1 || NT == 1, "columns of a row within one block");
    if constexpr (NC > 1) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[0][b][e] += nvk_dpp<NVK_DPP_QP_XOR1>(sc[0][b][e]);
    }
    if constexpr (NC > 2) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[0][b][e] += nvk_dpp<NVK_DPP_QP_XOR2>(sc[0][b][e]);
    }
    // finished here, and not behind the next branch: the lane exchanges would be moves of their own
    // there, and the products of every group be kept until then
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int b = 0; b < 4; ++b) asm volatile("" : "+v"(sc[t][b]));
    if (!last) issue_keys(at, kraw);

    // ---- mask, running maximum, probabilities
    const bool full = kbase + kCK - 1 <= full_limit;
    int seen[NT];  // of this lane's 16 keys, the first `seen`
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      nvk_f32x4(&c4)[4] = sc[t];
      seen[t] = row_limit[t] - kbase - 16 * g + 1;
      if (!full) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) c4[b][e] = 4 * b + e < seen[t] ? c4[b][e] : -INFINITY;
      }
      float mx = nvk_max3(nvk_max3(c4[0][0], c4[0][1], c4[0][2]),
                          nvk_max3(c4[0][3], c4[1][0], c4[1][1]),
                          nvk_max3(c4[1][2], c4[1][3], c4[2][0]));
      mx = nvk_max3(nvk_max3(c4[2][1], c4[2][2], c4[2][3]), mx,
                    nvk_max3(c4[3][0], c4[3][1], nvk_max3(c4[3][2], c4[3][3], c4[3][3])));
      mx = nvk_max_xor32(max_xor16(mx));
      const float m_new = fmaxf(m_run[t], mx * a.scale_log2);
      const float moff = m_new == -INFINITY ? 0.f : m_new;
      if (__builtin_amdgcn_ballot_w64(m_new > m_run[t])) {
        const float alpha = nvk_fast_exp2(m_run[t] - moff);  // 0 while nothing was visible
        l_part[t][0] *= alpha;
        l_part[t][1] *= alpha;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) acc[t][d] *= alpha;
        m_run[t] = m_new;
      }
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c4[b][e] = nvk_fast_exp2(fmaf(c4[b][e], a.scale_log2, -moff));
          l_part[t][e & 1] += c4[b][e];
        }
    }

    // ---- O^T += V^T (P vs)^T, one operand per group of dimensions
    vec8h pf[NT][NS][2];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      if (i < NS) {
        const auto* vp = scales(1, g0 + i);
        const nvk_u32x4 vs[2] = {__builtin_bit_cast(nvk_u32x4, vp[0]),
                                 __builtin_bit_cast(nvk_u32x4, vp[1])};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          nvk_u32x4 vm[2] = {vs[0], vs[1]};
          if (!full) {
            // a masked key's scale may be anything, what an earlier owner of the page left too
#pragma unroll
            for (int p = 0; p < 8; ++p) {
              const int n_seen = seen[t] - 2 * p;
              vm[p >> 2][p & 3] &= n_seen >= 2 ? 0xffffffffu : n_seen == 1 ? 0xffffu : 0u;
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            nvk_u32x4 x;
#pragma unroll
            for (int p = 0; p < 4; ++p)
              x[p] = times_scales(sc[t][2 * h + (p >> 1)][2 * (p & 1)],
                                  sc[t][2 * h + (p >> 1)][2 * (p & 1) + 1], vm[h][p]);
            pf[t][i][h] = __builtin_bit_cast(vec8h, x);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int d = 2 * i + h;
        const i32x2 vc = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(size_t)(buf + tr_row + 16 * (i ^ sw) +
                                                                8 * h));
#pragma unroll
        for (int k8 = 0; k8 < 2; ++k8) {
          const vec8h vf = fp4_unpack<true>((uint32_t)vc[k8]);
#pragma unroll
          for (int t = 0; t < NT; ++t)
            acc[t][d] = NvkElt<true>::mfma16x16x32(vf, pf[t][i % NS][k8], acc[t][d]);
        }
      }
      if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
    }

    if (!last) {
      wait_reads();
      issue_rest(at);
    }

    // ---- the group's or the range's end
    cut = last && !group_end;
    if (WHOLE) {
      ++k;
      continue;
    }
    if (group_end || last) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float l_tot = nvk_sum_xor32(sum_xor16(l_part[t][0] + l_part[t][1]));
        nvk_f32x4 o[kKeep];
        kept(o, t);
        if (group_end && started_here) {
          put_rows(o, l_tot, t);
        } else if (!started_here && wave > 0) {
#pragma unroll
          for (int j = 0; j < kKeep; ++j) s_o[wave - 1][t * kKeep + j][lane] = o[j];
          s_ml[wave - 1][t][lane] = make_float2(m_run[t], l_tot);
          if (lane == 0) s_ended[wave - 1] = group_end;
        } else if (group_end) {
          put_record(o, m_run[t], l_tot, t);
        }
      }
      if (lane == 0) {
        const int first = Hkv * s_cs[s] + (kvh * tiles + tile) * n;
        const int64_t e = ((int64_t)s * Hkv + kvh) * a.max_tiles + tile;
        *reinterpret_cast<int2*>(a.desc + 2 * e) =
            make_int2(sp.owner(first) / W, sp.owner(first + n - 1) / W);
      }
      if (last) break;
      s = ns;
      sq = nsq;
      kvh = nkvh;
      tile = ntile;
      n = nn;
      tiles = ntiles;
      k = 0;
      started_here = true;
      start_group();
    } else {
      ++k;
    }
  }

  if constexpr (!WHOLE) {
    // A group that is cut between waves of the workgroup: the first of them joins what the others hold.
    __syncthreads();
    if (!cut || (!started_here && wave > 0)) return;
    bool ended = false;
    nvk_f32x4 o[NT][kKeep];
    float l[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] = nvk_sum_xor32(sum_xor16(l_part[t][0] + l_part[t][1]));
      kept(o[t], t);
    }
    for (int v = wave + 1; v < W && !ended; ++v) {
      ended = uniform(s_ended[v - 1]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 ml = s_ml[v - 1][t][lane];
        const float m = fmaxf(m_run[t], ml.x), mref = m == -INFINITY ? 0.f : m;
        const float w0 = nvk_fast_exp2(m_run[t] - mref), w1 = nvk_fast_exp2(ml.x - mref);
        m_run[t] = m;
        l[t] = l[t] * w0 + ml.y * w1;
#pragma unroll
        for (int j = 0; j < kKeep; ++j) o[t][j] = o[t][j] * w0 + s_o[v - 1][t * kKeep + j][lane] * w1;
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
      if (started_here && ended)
        put_rows(o[t], l[t], t);
      else
        put_record(o[t], m_run[t], l[t], t);
  } else {
    // Wave v's rows to LDS (the values' buffers, used up): O, m, l; then a thread sums 4 dimensions of
    // a row over the waves.
    static_assert(NT == 1, "rows of one block");
    float* st = reinterpret_cast<float*>(lds);
    const float l_tot = nvk_sum_xor32(sum_xor16(l_part[0][0] + l_part[0][1]));
    nvk_f32x4 o[kKeep];
    kept(o, 0);
    wait_reads();
    __syncthreads();
    if (row_valid[0]) {
      float* rec = st + (wave * (kR / NC) + row) * kRec;
#pragma unroll
      for (int j = 0; j < kKeep; ++j) *reinterpret_cast<nvk_f32x4*>(rec + d0 + 16 * j) = o[j];
      if (g == 0 && g0 == 0) {
        rec[HD] = m_run[0];
        rec[HD + 1] = l_tot;
      }
    }
    __syncthreads();
    const int d = 4 * (tid % (HD / 4)), rows = min(sq.queries * a.G - tile * kR, kR / NC);
    for (int mrow = tid / (HD / 4); mrow < rows; mrow += 64 * W / (HD / 4)) {
      float M = -INFINITY;
#pragma unroll
      for (int v = 0; v < W; ++v) M = fmaxf(M, st[(v * (kR / NC) + mrow) * kRec + HD]);
      const float mref = M == -INFINITY ? 0.f : M;
      float L = 0.f;
      nvk_f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < W; ++v) {
        const float* rec = st + (v * (kR / NC) + mrow) * kRec;
        const float wt = nvk_fast_exp2(rec[HD] - mref);
        L += rec[HD + 1] * wt;
        O += wt * *reinterpret_cast<const nvk_f32x4*>(rec + d);
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;
      const int rr = tile * kR + mrow;
      const int mt = a.G == 1 ? rr : (int)__umulhi((uint32_t)rr, a.g_inverse);
      nvk_u32x2 wv;
      wv.x = E::pack2(O[0] * inv, O[1] * inv);
      wv.y = E::pack2(O[2] * inv, O[3] * inv);
      *reinterpret_cast<nvk_u32x2*>(a.out + (int64_t)(sq.row0 + mt) * a.out_stride_tok +
                                    (int64_t)(kvh * a.G + rr - mt * a.G) * a.out_stride_head +
                                    d) = wv;
    }
  }
}

// Merges the records of groups cut between waves and writes the rows of groups without a key.
// grid = (max_tiles * row pairs of a tile, Hkv, batch), W waves: a workgroup owns two rows of a group
// (HD / 4 lanes each, HD 64: half of them idle), wave v folds parts p1 + v, p1 + v + W, ... and wave 0
// joins the waves' states through LDS.
template <int HD, bool F16, int W>
__global__ __launch_bounds__(64 * W) void fp4_merge_kernel(AttnArgs a) {
  using E = NvkElt<F16>;
  constexpr int kRec = HD + 4, kLanes = HD / 4, kBatch = 4;
  const int pairs = (a.rec_rows + 1) / 2;
  const int tile = a.max_tiles == 1 ? 0 : blockIdx.x / pairs;
  const int pair = blockIdx.x - tile * pairs;
  const int kvh = blockIdx.y, s = blockIdx.z;
  const int lane = threadIdx.x & 63, v = uniform(threadIdx.x >> 6);
  const int64_t e = ((int64_t)s * a.num_kv_heads + kvh) * a.max_tiles + tile;
  int2 desc = *reinterpret_cast<const int2*>(a.desc + 2 * e);
  int row0 = s * a.n_query, queries = a.n_query;
  if (a.cu_q) {
    const Seq sq = seq_of(a, s);
    row0 = sq.row0;
    queries = sq.queries;
  }
  const int rows = min(queries * a.G - tile * a.tile_rows, a.rec_rows);  // of this tile
  if (2 * pair >= rows) return;
  const int p1 = desc.x, p2 = desc.y;
  if (p1 >= 0 && p1 == p2) return;  // finished by one workgroup
  const int half = lane / kLanes, d0 = 4 * (lane % kLanes);
  const bool ok = half < 2 && 2 * pair + half < rows;
  const int row = ok ? 2 * pair + half : 2 * pair;
  float M = -INFINITY, L = 0.f;
  nvk_f32x4 O = {0.f, 0.f, 0.f, 0.f};
  if (p1 >= 0) {
    for (int base = p1 + v; base <= p2; base += kBatch * W) {
      float mv[kBatch], lv[kBatch];
      nvk_f32x4 ov[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        // past the last part: it is read again, and replaced (a branch around each load would wait
        // for it there, one after the other)
        const int p = min(base + u * W, p2);
        const float* rec =
            a.rec + (((int64_t)p * 2 + (p == p1 ? 0 : 1)) * a.rec_rows + row) * kRec;
        const float2 ml = *reinterpret_cast<const float2*>(rec + HD);
        mv[u] = ml.x;
        lv[u] = ml.y;
        ov[u] = *reinterpret_cast<const nvk_f32x4*>(rec + d0);
      }
#pragma unroll
      for (int u = 1; u < kBatch; ++u) {
        const bool part = base + u * W <= p2;
        mv[u] = part ? mv[u] : -INFINITY;
        lv[u] = part ? lv[u] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ov[u][i] = part ? ov[u][i] : 0.f;
      }
      float mb = M;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) mb = fmaxf(mb, mv[u]);
      const float mref = mb == -INFINITY ? 0.f : mb;
      const float rs = nvk_fast_exp2(M - mref);
      L *= rs;
      O *= rs;
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float wt = nvk_fast_exp2(mv[u] - mref);
        L += lv[u] * wt;
        O += wt * ov[u];
      }
      M = mb;
    }
  }
  if constexpr (W > 1) {
    __shared__ float sm[W][64], sl[W][64];
    __shared__ nvk_f32x4 so[W][64];
    sm[v][lane] = M;
    sl[v][lane] = L;
    so[v][lane] = O;
    __syncthreads();
    if (v != 0) return;
    float mx = M;
#pragma unroll
    for (int i = 1; i < W; ++i) mx = fmaxf(mx, sm[i][lane]);
    const float mref = mx == -INFINITY ? 0.f : mx;
    L = 0.f;
    O = nvk_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float wt = nvk_fast_exp2(sm[i][lane] - mref);
      L += sl[i][lane] * wt;
      O += wt * so[i][lane];
    }
  }
  if (!ok) return;
  const int rr = tile * a.tile_rows + row;
  const int tok = rr / a.G, head = kvh * a.G + rr - tok * a.G;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  nvk_u32x2 wv;
  wv.x = E::pack2(O[0] * inv, O[1] * inv);
  wv.y = E::pack2(O[2] * inv, O[3] * inv);
  *reinterpret_cast<nvk_u32x2*>(a.out + (int64_t)(row0 + tok) * a.out_stride_tok +
                                (int64_t)head * a.out_stride_head + d0) = wv;
}

// Sizes that follow from a call's static bounds.
struct Plan {
  int tile_rows, max_tiles, rec_rows, n_waves, wave_shift;
  size_t desc_bytes, bytes;
};
// Tiles of 32 rows: a chunk takes a wave half as long again as with 16, for twice the rows.  That gains
// where every wave has several chunks, and loses where twice as many tiles share the CUs better.
// Measured, tiles of 16 / 32 rows, 16/8 heads and (chunks of 32-row tiles per wave, by the table's
// width):
//   32 x 9 queries over U{1024..8192} (16) 72.1 / 64.2 us, 32 x 32 (32) 132 / 114, 32 x 64 (64) 251 / 211;
//   16/16 heads, 16 x 20 over U{2000..4000} (8) 55.1 / 49.7; 16/2 heads, 32 x 16 (8) 55.0 / 51.5; 4 x 64
//   over 8000 (8) 58.4 / 54.1;
//   4 x 32 over 8000 (4) 36.4 / 35.2; 16/2 heads, 16 x 16 over U{2000..4000} (4) 36.1 / 37.2; 1 x 64 over
//   8000 (2) 24.1 / 27.7, 16/2 heads, 8 x 16 over 2000 (1) 19.5 / 21.6, 1 x 64 over 100 (less) 9.4 / 12.0.
// An odd number of 16-row blocks leaves half a tile empty, which 7 are enough to make up for (64 x 100
// queries, 13 blocks, 206 / 170; 32 x 12, 16/4 heads, 3 blocks, over U{500..4000} 37.6 / 37.5; 5 blocks: 32
// x 20, 16/4 heads, 51.9 / 53.9, 32 x 40 160 / 158).
bool wide_tiles(int64_t rows, int64_t chunks) {
  const int64_t blocks = (rows + kR - 1) / kR, tiles = (blocks + 1) / 2;
  return (blocks % 2 == 0 || blocks >= 7) && tiles <= INT32_MAX / (chunks < 1 ? 1 : chunks) &&
         tiles * chunks >= 6 * kMaxWGs * kWavesPerWG;
}

// What either route takes.
bool sizes_ok(int batch, int max_queries, int num_q_heads, int num_kv_heads, int head_dim,
              int block_size, int max_blocks) {
  if (batch <= 0 || batch > kMaxBatch || max_queries <= 0 || num_q_heads <= 0 ||
      num_kv_heads <= 0 || num_q_heads % num_kv_heads || block_size <= 0 || max_blocks <= 0)
    return false;
  if ((head_dim != 128 && head_dim != 64) || block_size % 16) return false;
  const int G = num_q_heads / num_kv_heads;
  return G <= kR && num_kv_heads <= 65535 && (int64_t)max_queries * G < 1 << 27 &&
         (int64_t)max_blocks * block_size <= INT32_MAX - kCK &&
         (int64_t)block_size * num_kv_heads * head_dim <= INT32_MAX;
}

// Of sizes that are ok.  False: more (tile, chunk) pairs than the split counts in 32 bits.
bool plan_of(int batch, int max_queries, int num_q_heads, int num_kv_heads, int head_dim,
             int block_size, int max_blocks, Plan& p) {
  const int64_t rows = (int64_t)max_queries * (num_q_heads / num_kv_heads);
  const int64_t chunks = ((int64_t)max_blocks * block_size + kCK - 1) / kCK;
  p.tile_rows = wide_tiles(rows, chunks * batch * num_kv_heads) ? 2 * kR : kR;
  const int64_t tiles = (rows + p.tile_rows - 1) / p.tile_rows;
  if (tiles * chunks > INT32_MAX / batch / num_kv_heads) return false;
  p.max_tiles = (int)tiles;
  p.rec_rows = (int)(rows < p.tile_rows ? rows : p.tile_rows);
  const int64_t units = tiles * chunks * batch * num_kv_heads;
  p.wave_shift = 2;  // a workgroup's
  while ((1 << p.wave_shift) < units && (1 << p.wave_shift) < kMaxWGs * kWavesPerWG) ++p.wave_shift;
  p.n_waves = 1 << p.wave_shift;
  p.desc_bytes = ((size_t)batch * num_kv_heads * tiles * 8 + 255) / 256 * 256;
  p.bytes = p.desc_bytes + (size_t)p.n_waves / kWavesPerWG * 2 * p.rec_rows * (head_dim + 4) *
                               sizeof(float);
  return true;
}

// Waves of a workgroup that takes a group by itself (WHOLE; 0: ranges): one kernel, no records, and all
// of a group's chunks on their way at once, but a CU's time is that of the groups that fall to it.  By
// the number of groups (a CU holds 2 to 4 such workgroups) and the most keys that one can have.  16/8
// heads, ranges / 4 waves / 8 waves:
//   up to 256 keys: 1 x 100 7.1 / 4.5 / 5.4 us, 64 x U{16..256} 11.1 / 7.3 / 7.9, 512 x U{16..256} 29.1 /
//   23.0 / 38.5, 4 x 16 queries over 256 10.0 / 6.2 / 7.4, 64 x 96 over U{100..250} 57 / 50 / 127;
//   up to 1024: 1 x 1000 8.4 / 8.5 / 7.5, 32 x U{100..1024} (256 groups) 13.9 / 11.0 / 9.8, 64 (512) 16.9 /
//   14.2 / 14.4, 256 (2048) 37.5 / 34.8 / 37.3, 32 x 6 queries 19.2 / 13.2 / 11.9, 64 x 6 22.9 / 17.5 /
//   20.5, 32 x 64 queries (2048) 47 / 42 / 66, 64 x 64 over U{600..1000} (4096) 88 / 93 / 149;
//   up to 2048, ranges / 8 waves: 4 x 2048 (32) 9.7 / 12.4, but called one by one 15.7 / 12.7 (the second
//   kernel is 3 us of the host's); 8 x 2048 (64) 11.8 / 12.5, 16 x U{100..2048} 14.6 / 13.1, 32 x 16.9 /
//   14.3, 64 x 22.3 / 19.5, 64 x 2048 32.0 / 30.5, 128 x U{100..2048} (1024) 36.1 / 34.5; 6 queries: 32 x
//   U{100..2048} 22.8 / 17.3, 48 x (384) 26.4 / 27.3;
//   up to 4096: 32 x U{100..4096} 23.4 / 23.1, 32 x 4096 32.8 / 29.3, 16 x 4096 (128) 20.1 / 23.0, 48 x
//   U{100..4096} (384) 28.6 / 35.7; up to 8192: 32 x U{100..8192} 35.5 / 40.9.
constexpr int kCUs = 256;
int whole_waves(int rows, int head_dim, int64_t groups, int64_t max_keys) {
  if (rows > 65535) return 0;  // tiles along a grid's z
  if (max_keys <= 1024) {
    if (groups * ((max_keys + kCK - 1) / kCK) >= 65536) return 0;
    return max_keys > 256 && groups <= kCUs ? 8 : 4;
  }
  const bool few = rows <= kR / (head_dim / kFp4Group);
  if (max_keys <= 2048) return groups >= kCUs / 8 && groups <= (few ? 4 : 1) * kCUs ? 8 : 0;
  return max_keys <= 4096 && groups >= kCUs * 3 / 4 && groups <= kCUs ? 8 : 0;
}

template <int HD, bool F16>
int launch(const AttnArgs& a, int max_keys, hipStream_t s) {
  constexpr int NG = HD / kFp4Group;
  const dim3 grid(a.n_waves / kWavesPerWG), block(64 * kWavesPerWG);
  const int rows = a.n_query * a.G;
  const std::integral_constant<int, 1> c1;
  const std::integral_constant<int, 2> c2;
  const std::integral_constant<int, NG> few;
  const std::integral_constant<int, 4> four;
  const std::integral_constant<int, 8> eight;
  const int tiles16 = (rows + kR - 1) / kR;
  if (const int w =
          whole_waves(rows, HD, (int64_t)a.batch * a.num_kv_heads * tiles16, max_keys)) {
    AttnArgs b = a;
    const bool deal = (int64_t)a.batch * a.num_kv_heads > kCUs && tiles16 == 1 &&
                      a.batch <= kBalanced && a.num_kv_heads <= kCUs && max_keys > 512;
    b.round = deal ? kCUs / a.num_kv_heads : 0;
    const auto one_kernel = [&](auto nc, auto waves) {
      constexpr int NC = decltype(nc)::value, W = decltype(waves)::value;
      const dim3 groups(a.num_kv_heads, a.batch, tiles16);
      if (a.block_size % kCK)
        hipLaunchKernelGGL((fp4_attention_kernel<HD, F16, false, NC, 1, W, true>), groups,
                           dim3(64 * W), 0, s, b);
      else
        hipLaunchKernelGGL((fp4_attention_kernel<HD, F16, true, NC, 1, W, true>), groups,
                           dim3(64 * W), 0, s, b);
    };
    const auto by_rows = [&](auto waves) {
      if (rows <= kR / NG) one_kernel(few, waves);
      else if (rows <= kR / 2) one_kernel(c2, waves);
      else one_kernel(c1, waves);
    };
    w == 4 ? by_rows(four) : by_rows(eight);
    return nvk_launch_status();
  }
  const auto main = [&](auto nc, auto nt) {
    constexpr int NC = decltype(nc)::value, NT = decltype(nt)::value;
    if (a.block_size % kCK)
      hipLaunchKernelGGL((fp4_attention_kernel<HD, F16, false, NC, NT>), grid, block, 0, s, a);
    else
      hipLaunchKernelGGL((fp4_attention_kernel<HD, F16, true, NC, NT>), grid, block, 0, s, a);
  };
  if (rows <= kR / NG) main(few, c1);
  else if (rows <= kR / 2) main(c2, c1);
  else if (a.tile_rows == kR) main(c1, c1);
  else main(c1, c2);
  const int st = nvk_launch_status();
  if (st != NVK_OK) return st;
  const dim3 mgrid(a.max_tiles * ((a.rec_rows + 1) / 2), a.num_kv_heads, a.batch);
  // By the parts that a group has on average, where it has any: a wave fetches 4 in a round trip.
  // One wave / four per row pair, 16/8 heads: 16/2 heads, 8 x 16 queries over 2000 (4 parts) 18.3 / 18.9
  // us; 8 x 1 over 4000 (8) 14.7 / 14.4, 4 over U{8192..32768} (16) 28.5 / 26.6; four / sixteen: 2 over
  // 16000 (32) 15.3 / 15.4, 1 over 30000 (64) 16.3 / 15.2, 8/1 heads, 1 over 100000 (512) 27.4 / 19.7.
  const int64_t parts =
      a.n_waves / kWavesPerWG / ((int64_t)a.batch * a.num_kv_heads * a.max_tiles);
  if (parts >= 32)
    hipLaunchKernelGGL((fp4_merge_kernel<HD, F16, 16>), mgrid, dim3(64 * 16), 0, s, a);
  else if (parts >= 8)
    hipLaunchKernelGGL((fp4_merge_kernel<HD, F16, 4>), mgrid, dim3(64 * 4), 0, s, a);
  else
    hipLaunchKernelGGL((fp4_merge_kernel<HD, F16, 1>), mgrid, dim3(64), 0, s, a);
  return nvk_launch_status();
}

// Long query ranges go through f16 pages (fp4.h).
// From 193 rows (queries x G) per kv head on, where the step has work for more than that route's three
// or four kernels: 16384 chunks of 64 keys under tiles of 16 rows.  Measured, the kernel above / pages,
// 16/8 heads:
//   128 rows: 32 x 64 queries over U{1024..8192} 194 / 345 us, 1 x 64 over 8000 23.5 / 36.3; 192: 281 / 421,
//   29.4 / 35.9, 16/16 heads, 16 x 192 over U{2000..4000} 201 / 254; 200: 64 x 100 over U{600..1500} 170 /
//   184, 16 x 100 63 / 58; 240: 32 x 120 110 / 88; 256: 32 x 128 over U{1024..8192} 371 / 424; 384: 565 / 557;
//   by the chunks: 1 x 512 over 512 (4096) 11.7 / 19.9, 4 x 256 over 300 (5120) 15.8 / 19.1, 16 x 128 over
//   256 (8192) 20.6 / 24.9, 8 x 200 over 500 (12800) 26.6 / 28.8, 1 x 1000 over 1000 (16000) 28.0 / 30.2,
//   4 x 512 over 512 (16384) 30.4 / 24.7, 32 x 128 over 256 (16384) 37.5 / 33.8.
constexpr int kDirectRows = 192;
constexpr int64_t kDirectChunks = 16384;
constexpr int64_t kPageBytesMost = (int64_t)512 << 20;  // pages of a part of the batch (one sequence: any)

// Workspace of that route, for `part` sequences at a time.
struct PagePlan {
  int part, pages_per_seq, max_keys;
  size_t cu_bytes, table_bytes, page_bytes, attn_bytes, bytes;  // page_bytes: of keys, and of values
};
bool page_plan(int batch, int max_queries, int max_seqlen_k, int num_q_heads, int num_kv_heads,
               int head_dim, int block_size, int max_blocks, PagePlan& p) {
  const int G = num_q_heads / num_kv_heads;
  if (head_dim != 128 || (G != 1 && G != 2 && G != 4 && G != 8) ||
      (int64_t)max_queries * G <= kDirectRows)
    return false;
  int64_t keys = (int64_t)max_blocks * block_size;
  if (max_seqlen_k > 0 && max_seqlen_k < keys) keys = max_seqlen_k;
  const int64_t tiles = ((int64_t)max_queries * G + kR - 1) / kR, chunks = (keys + kCK - 1) / kCK;
  if (tiles * chunks < kDirectChunks && tiles * chunks * batch * num_kv_heads < kDirectChunks)
    return false;
  if ((int64_t)num_kv_heads * head_dim >= (1 << 23) ||
      (int64_t)kFp4Page * num_kv_heads * head_dim * 2 > UINT32_MAX || num_kv_heads > 65535 ||
      (int64_t)max_queries * G > 65535 * (int64_t)128)
    return false;
  p.max_keys = (int)keys;
  p.pages_per_seq = (int)((keys + kFp4Page - 1) / kFp4Page);
  const int64_t per_seq = (int64_t)p.pages_per_seq * kFp4Page * num_kv_heads * head_dim * 2;
  const int64_t fit = kPageBytesMost / (2 * per_seq);
  p.part = (int)(fit < 1 ? 1 : fit < batch ? fit : batch);
  if ((int64_t)p.part * p.pages_per_seq > INT32_MAX) return false;
  const auto pad = [](size_t x) { return (x + 255) / 256 * 256; };
  p.cu_bytes = pad((size_t)2 * (batch + 1) * sizeof(int32_t));
  p.table_bytes = pad((size_t)p.part * p.pages_per_seq * sizeof(int32_t));
  p.page_bytes = (size_t)p.part * per_seq;
  p.attn_bytes = pad(nvk_varlen_prefill_parts_workspace_size(p.part, max_queries, p.max_keys,
                                                             num_q_heads, num_kv_heads, head_dim));
  // the last part of the batch may be smaller, and cut its tiles into more parts
  const int rest = batch % p.part;
  if (rest) {
    const size_t r = pad(nvk_varlen_prefill_parts_workspace_size(
        rest, max_queries, p.max_keys, num_q_heads, num_kv_heads, head_dim));
    p.attn_bytes = r > p.attn_bytes ? r : p.attn_bytes;
  }
  p.bytes = p.cu_bytes + p.table_bytes + 2 * p.page_bytes + p.attn_bytes;
  return true;
}

int launch_pages(const AttnArgs& a, const PagePlan& p, int num_q_heads, float scale, bool f16,
                 void* workspace, hipStream_t s) {
  char* at = static_cast<char*>(workspace);
  const int32_t *cu_q = a.cu_q, *cu_k = a.keys;
  Fp4Expand e{};
  if (!cu_q) {  // the same number of queries each: the first pass makes the prefix sums as well
    e.lens = a.keys;
    e.total_batch = a.batch;
    e.n_query = a.n_query;
    e.cu_q_out = reinterpret_cast<int32_t*>(at);
    e.cu_k_out = e.cu_q_out + a.batch + 1;
    cu_q = e.cu_q_out;
    cu_k = e.cu_k_out;
  }
  at += p.cu_bytes;
  e.tables = reinterpret_cast<int32_t*>(at);
  at += p.table_bytes;
  e.k_pages = reinterpret_cast<uint16_t*>(at);
  at += p.page_bytes;
  e.v_pages = reinterpret_cast<uint16_t*>(at);
  at += p.page_bytes;
  e.k_data = a.k_data;
  e.v_data = a.v_data;
  e.k_scale = a.k_scale;
  e.v_scale = a.v_scale;
  e.bt_stride = a.bt_stride;
  e.pages_per_seq = p.pages_per_seq;
  e.max_blocks = a.cap / a.block_size;
  e.block_size = a.block_size;
  e.bs_shift = a.bs_shift;
  e.num_blocks = a.num_blocks;
  e.num_kv_heads = a.num_kv_heads;
  e.f16 = f16;
  Fp4Prefill f{};
  f.q = a.q;
  f.q_stride_tok = a.q_stride_tok;
  f.q_stride_head = a.q_stride_head;
  f.total_q = a.total_q;
  f.k_pages = e.k_pages;
  f.v_pages = e.v_pages;
  f.tables = e.tables;
  f.max_seqlen_q = a.n_query;
  f.max_seqlen_k = p.max_keys;
  f.pages_per_seq = p.pages_per_seq;
  f.num_q_heads = num_q_heads;
  f.num_kv_heads = a.num_kv_heads;
  f.scale = scale;
  f.out = a.out;
  f.out_stride_tok = a.out_stride_tok;
  f.out_stride_head = a.out_stride_head;
  f.workspace = at;
  f.workspace_bytes = p.attn_bytes;
  f.f16 = f16;
  for (int b = 0; b < a.batch; b += p.part) {
    e.batch = f.batch = a.batch - b < p.part ? a.batch - b : p.part;
    e.block_tables = a.block_tables + b * a.bt_stride;
    e.cu_k = f.cu_k = cu_k + b;
    f.cu_q = cu_q + b;
    e.first = b;
    int st = fp4_expand_launch(e, s);
    e.cu_q_out = e.cu_k_out = nullptr;
    if (st == NVK_OK) st = fp4_prefill_launch(f, s);
    if (st != NVK_OK) return st;
  }
  return NVK_OK;
}

}  // namespace

extern "C" size_t nvk_fp4_attention_workspace_size(int32_t batch, int32_t max_seqlen_q,
                                                   int32_t max_seqlen_k, int32_t num_q_heads,
                                                   int32_t num_kv_heads, int32_t head_dim,
                                                   int32_t block_size, int32_t max_blocks) {
  Plan p;
  PagePlan pp;
  if (!sizes_ok(batch, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks))
    return 0;
  if (page_plan(batch, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads, head_dim, block_size,
                max_blocks, pp))
    return pp.bytes;
  return plan_of(batch, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks, p)
             ? p.bytes
             : 0;
}

extern "C" int nvk_fp4_attention(const void* q, int64_t q_stride_tok, int64_t q_stride_head,
                                 int64_t total_q, const void* k_data, const void* k_scale,
                                 const void* v_data, const void* v_scale,
                                 const int32_t* cu_seqlens_q, const int32_t* seqlens_k,
                                 int32_t batch, int32_t max_seqlen_q, int32_t max_seqlen_k,
                                 const int32_t* block_tables, int64_t bt_stride,
                                 int32_t max_blocks, int32_t block_size, int32_t num_blocks,
                                 int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                 float scale, void* out, int64_t out_stride_tok,
                                 int64_t out_stride_head, void* workspace, size_t workspace_bytes,
                                 int32_t dtype, void* stream) {
  if (batch < 0 || total_q < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      block_size <= 0 || max_blocks < 0 || num_blocks < 0 || num_q_heads % num_kv_heads)
    return NVK_EINVAL;
  if (!(scale > 0.f)) return NVK_EINVAL;
  if (dtype != NVK_DTYPE_BF16 && dtype != NVK_DTYPE_F16) return NVK_EUNSUPPORTED;
  if (batch == 0 || total_q == 0 || max_seqlen_q == 0) return NVK_OK;
  if (total_q > INT32_MAX) return NVK_EINVAL;
  if (!cu_seqlens_q && (int64_t)batch * max_seqlen_q != total_q) return NVK_EINVAL;
  Plan p{};
  PagePlan pp;
  if (num_blocks == 0 || !sizes_ok(batch, max_seqlen_q, num_q_heads, num_kv_heads, head_dim,
                                   block_size, max_blocks))
    return NVK_EUNSUPPORTED;
  const bool pages = page_plan(batch, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads,
                               head_dim, block_size, max_blocks, pp);
  if (!pages && !plan_of(batch, max_seqlen_q, num_q_heads, num_kv_heads, head_dim, block_size,
                         max_blocks, p))
    return NVK_EUNSUPPORTED;
  if (!q || !k_data || !k_scale || !v_data || !v_scale || !seqlens_k || !block_tables || !out)
    return NVK_EINVAL;
  if (bt_stride < max_blocks) return NVK_EINVAL;
  if (((uintptr_t)q | (uintptr_t)k_data | (uintptr_t)k_scale | (uintptr_t)v_data |
       (uintptr_t)v_scale) % 16 || q_stride_tok % 8 || q_stride_head % 8)
    return NVK_EALIGN;
  if ((uintptr_t)out % 8 || out_stride_tok % 4 || out_stride_head % 4) return NVK_EALIGN;
  if (((uintptr_t)cu_seqlens_q | (uintptr_t)seqlens_k | (uintptr_t)block_tables) % 4)
    return NVK_EALIGN;
  if (!workspace || workspace_bytes < (pages ? pp.bytes : p.bytes)) return NVK_EWORKSPACE;
  if ((uintptr_t)workspace % 256) return NVK_EALIGN;
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride_tok = q_stride_tok;
  a.q_stride_head = q_stride_head;
  a.total_q = total_q;
  a.k_data = static_cast<const uint8_t*>(k_data);
  a.k_scale = static_cast<const uint16_t*>(k_scale);
  a.v_data = static_cast<const uint8_t*>(v_data);
  a.v_scale = static_cast<const uint16_t*>(v_scale);
  a.cu_q = cu_seqlens_q;
  a.keys = seqlens_k;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.batch = batch;
  a.n_query = max_seqlen_q;
  a.tile_rows = p.tile_rows;
  a.max_tiles = p.max_tiles;
  a.cap = max_blocks * block_size;
  a.block_size = block_size;
  a.bs_shift = nvk_log2_exact(block_size);
  a.num_blocks = num_blocks;
  a.num_kv_heads = num_kv_heads;
  a.G = num_q_heads / num_kv_heads;
  a.g_inverse = a.G > 1 ? (uint32_t)((((uint64_t)1 << 32) + a.G - 1) / a.G) : 0;
  a.scale_log2 = scale * NVK_LOG2E;
  a.out = static_cast<uint16_t*>(out);
  a.out_stride_tok = out_stride_tok;
  a.out_stride_head = out_stride_head;
  a.desc = static_cast<int32_t*>(workspace);
  a.rec = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.desc_bytes);
  a.rec_rows = p.rec_rows;
  a.n_waves = p.n_waves;
  a.wave_shift = p.wave_shift;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool f16 = dtype == NVK_DTYPE_F16;
  if (pages) return launch_pages(a, pp, num_q_heads, scale, f16, workspace, s);
  const int max_keys = max_seqlen_k > 0 && max_seqlen_k < a.cap ? max_seqlen_k : a.cap;
  if (head_dim == 128)
    return f16 ? launch<128, true>(a, max_keys, s) : launch<128, false>(a, max_keys, s);
  return f16 ? launch<64, true>(a, max_keys, s) : launch<64, false>(a, max_keys, s);
}
