// Attention of each sequence's new tokens over the paged cache
// (ncm_tree_attention): one decoded token, or a chain or tree of drafted ones.
//
//   out = sum_k p_k v_k / sum_k p_k,  p_k = 2^(t_k - m),  t_k = log2(e) scale q.k
//
// The query rows of one kv head (its heads / kv_heads query heads of every
// node) form tiles of up to ROWS rows; an item is (sequence, kv head, tile).
// A CTA holds KG key groups of RG warps. A key group takes every KG-th tile of
// 32 keys through a cp.async ring of its own (zero-filled behind the last
// key), its warps each hold 16 MT query rows in registers: S = Q K^T and P V
// are m16n8k16 products with f32 sums, P never leaves the registers, and codes
// become bf16 in registers (both code types are exact in bf16; a key's scale
// multiplies its score, a value's scale its probability). The maximum m is
// only moved when a score passes it by 2^8, so most tiles neither reduce over
// lanes nor rescale. The key groups' sums meet in shared memory at the end.
//
// Split: items are cut into units of unit_keys keys, and every CTA of one wave
// takes the same number of consecutive units, whatever the sequences' lengths
// are (they are known on the device only). A CTA that ends inside an item
// leaves its sums in the workspace: slot 2c for an item begun by an earlier
// CTA, slot 2c + 1 for one that goes on in the next. merge_kernel adds the
// slots of such items up, in order.
//
// Order of contractions: the m16n8k16 products sum over head_dim in any order,
// so a lane reads 16 consecutive bytes of a key, and Q's fragments are
// permuted to match (lane % 4 = c holds the same dims of Q and K).
#include <algorithm>

#include "kv_cache.cuh"

namespace ncm {
namespace {

constexpr int kTile = 32;        // keys of one ring stage
constexpr float kFirstMax = -1e30f;
constexpr float kSlack = 8.f;    // scores may pass the running maximum by 2^8

struct TreeArgs {
  KvPools pools;
  KvBatch batch;
  const uint16_t* q;
  long long q_stride;
  const uint32_t* mask;
  int mask_words;
  int heads, group, max_nodes;
  float scale_log2;
  uint16_t* out;
  long long out_stride;
  float* lse;
  float* part;  // [2 * grid][ROWS][2 + HD]: maximum, sum, values
  int unit_keys;
  int grid;  // CTAs of the attention kernel
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// 16 (4) bytes from global to shared memory, zeros where !live.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

__device__ __forceinline__ uint32_t sub_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Bytes I and J of w as two bf16 values, exactly. int8: 128 + (low seven bits) minus
// 128 or 256, by the sign bit. e4m3: the code's exponent and mantissa moved into
// bf16's fields are the value times 2^-120 (subnormal codes included).
template <int FMT, int I, int J>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  if constexpr (FMT == NCM_KV_INT8) {
    const uint32_t x = prmt(w, 0x43u, 0x4040u | I | (J << 8));  // bytes: I, 0x43, J, 0x43
    return sub_bf16x2(x & 0x437F437Fu, x & 0x43804380u);
  } else {
    const uint32_t x = prmt(w, 0u, 0x0404u | (I << 4) | (J << 12));  // bytes: 0, I, 0, J
    const uint32_t y = ((x & 0x7F007F00u) >> 4) | (x & 0x80008000u);
    return mul_bf16x2(y, 0x7B807B80u);  // 2^120
  }
}

__device__ __forceinline__ uint32_t pack_rn(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// What one sequence contributes: its nodes (0 where its numbers do not fit), keys and units.
struct Seq {
  int first, n, len;
};
__device__ __forceinline__ Seq load_seq(const TreeArgs& a, int b, bool report) {
  Seq s;
  s.first = __ldg(a.batch.token_start + b);
  s.n = __ldg(a.batch.token_start + b + 1) - s.first;
  s.len = __ldg(a.batch.kv_lens + b);
  const bool bad = s.first < 0 || s.n < 0 || s.n > a.max_nodes || s.len < s.n ||
                   static_cast<long long>(s.first) + s.n > a.batch.rows ||
                   s.len > (static_cast<long long>(a.batch.table_width) << a.pools.page_shift);
  if (bad) {
    if (report) atomicOr(a.err, kErrBadIndex);
    s.n = s.len = 0;
  }
  return s;
}

template <int ROWS>
__device__ __forceinline__ int tiles_of(const TreeArgs& a, const Seq& s) {
  return (s.n * a.group + ROWS - 1) / ROWS;
}
__device__ __forceinline__ int units_of(const TreeArgs& a, const Seq& s) { return (s.len + a.unit_keys - 1) / a.unit_keys; }

// Units in front of sequence `upto` (whole warps; every lane gets the sum).
template <int ROWS>
__device__ __forceinline__ long long units_before(const TreeArgs& a, int upto) {
  long long sum = 0;
  for (int b = threadIdx.x & 31; b < upto; b += 32) {
    const Seq s = load_seq(a, b, false);
    sum += static_cast<long long>(tiles_of<ROWS>(a, s)) * a.pools.kv_heads * units_of(a, s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// The sequence that holds unit x < total, and the unit's place in it.
template <int ROWS>
__device__ __forceinline__ int find_unit(const TreeArgs& a, long long x, long long* inside) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < a.batch.batch; b0 += 32) {
    long long u = 0;
    if (b0 + lane < a.batch.batch) {
      const Seq s = load_seq(a, b0 + lane, false);
      u = static_cast<long long>(tiles_of<ROWS>(a, s)) * a.pools.kv_heads * units_of(a, s);
    }
    long long before = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += y;
    }
    const long long all = __shfl_sync(0xffffffffu, before, 31);
    before -= u;
    if (x < all) {
      const unsigned hit = __ballot_sync(0xffffffffu, x >= before && x < before + u);
      const int who = __ffs(hit) - 1;
      *inside = x - __shfl_sync(0xffffffffu, before, who);
      return b0 + who;
    }
    x -= all;
  }
  *inside = 0;
  return a.batch.batch;
}

// Bits [j0, j0 + 32) of a node's mask row (bits in front of 0 are ones, behind the row zeros).
__device__ __forceinline__ uint32_t mask_window(const uint32_t* row, int words, int j0) {
  if (j0 <= -32) return 0xFFFFFFFFu;
  if (j0 < 0) {
    const uint32_t w = words > 0 ? __ldg(row) : 0u;
    return (w << -j0) | ((1u << -j0) - 1u);
  }
  const int i = j0 >> 5;
  const uint32_t lo = i < words ? __ldg(row + i) : 0u, hi = i + 1 < words ? __ldg(row + i + 1) : 0u;
  return __funnelshift_r(lo, hi, j0 & 31);
}
__device__ __forceinline__ uint32_t first_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

template <int HD, int FMT, int MT, int RG, int KG>
struct TreeShape {
  static constexpr int kThreads = 32 * RG * KG;
  static constexpr int kRows = 16 * MT * RG;
  static constexpr int kRowBytes = HD * (FMT == NCM_KV_BF16 ? 2 : 1);
  static constexpr int kStageBytes = 2 * kTile * kRowBytes + (FMT == NCM_KV_BF16 ? 0 : 2 * kTile * 4);
  // two tiles in flight beside the one in use
  static constexpr int kStages = 3;
  static constexpr int kRingBytes = KG * kStages * kStageBytes;
  static constexpr int kMergeBytes = KG * kRows * (HD + 4) * 4;
  static constexpr int kSmem = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;
};

// 16-byte piece `chunk` of key `key` in a stage: pieces are permuted so that the
// eight rows of an ldmatrix, and two neighbouring keys' first (or last) four
// pieces, lie in different banks.
template <int RB>
__device__ __forceinline__ uint32_t piece_at(int key, int chunk) {
  if constexpr (RB == 64)
    return key * RB + ((chunk ^ ((key >> 1) & 3)) << 4);
  else
    return key * RB + ((chunk ^ (((key & 1) << 2) | ((key >> 1) & 3))) << 4);
}

template <int HD, int FMT, int MT, int RG, int KG>
__global__ void __launch_bounds__(32 * RG * KG) tree_attention_kernel(const TreeArgs a) {
  using S = TreeShape<HD, FMT, MT, RG, KG>;
  constexpr int RB = S::kRowBytes, CPR = RB / 16, ROWS = S::kRows, NST = S::kStages;
  constexpr int KS = HD / 16;       // k-steps of S
  constexpr int WPC = FMT == NCM_KV_BF16 ? 2 : 4;  // k-steps in a 16-byte piece
  constexpr int DPC = FMT == NCM_KV_BF16 ? 8 : 16;  // dims in a 16-byte piece
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kg = warp / RG, rg = warp % RG;
  const int r = lane >> 2, c = lane & 3;
  const int gt = rg * 32 + lane;  // thread of the key group
  const uint32_t ring = smem_u32(smem) + kg * NST * S::kStageBytes;
  pdl_wait();
  pdl_launch_dependents();

  const long long total = units_before<ROWS>(a, a.batch.batch);
  const long long lo = total * blockIdx.x / a.grid, hi = total * (blockIdx.x + 1) / a.grid;
  if (blockIdx.x == 0 && warp == 0)
    for (int b = lane; b < a.batch.batch; b += 32) load_seq(a, b, true);
  if (lo >= hi) return;
  long long inside;
  int b = find_unit<ROWS>(a, lo, &inside);

  auto group_sync = [&] {
    if constexpr (RG == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + kg), "n"(32 * RG) : "memory");
  };

  for (long long at = lo; at < hi && b < a.batch.batch;) {
    Seq s = load_seq(a, b, false);
    int units = units_of(a, s);
    const int tiles = tiles_of<ROWS>(a, s);
    if (inside >= static_cast<long long>(units) * tiles * a.pools.kv_heads) {  // (empty sequences too)
      ++b;
      inside = 0;
      continue;
    }
    const int item = static_cast<int>(inside / units), u0 = static_cast<int>(inside - static_cast<long long>(item) * units);
    const int u1 = static_cast<int>(min(static_cast<long long>(units), u0 + (hi - at)));
    const int kvh = item / tiles, row0 = (item - kvh * tiles) * ROWS;
    const int ctx = s.len - s.n;
    const int key0 = u0 * a.unit_keys, key1 = static_cast<int>(min(static_cast<long long>(s.len), static_cast<long long>(u1) * a.unit_keys));
    const int live_rows = s.n * a.group - row0;  // rows of this tile that exist (may be more than ROWS)

    // ---- this warp's query rows, in fragment order
    uint32_t qf[MT][KS][4];
    int node[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = rg * 16 * MT + mt * 16 + r + 8 * e;
        const bool live = row < live_rows;
        const int i = live ? (row0 + row) / a.group : 0;
        const int head = kvh * a.group + (live ? (row0 + row) - i * a.group : 0);
        node[mt][e] = live ? i : -1;
        const uint16_t* src = a.q + (s.first + static_cast<long long>(i)) * a.q_stride + head * HD;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int d = ((ks / WPC) * 4 + c) * DPC + (ks % WPC) * 4;
          uint2 v = make_uint2(0u, 0u);
          if (live) v = *reinterpret_cast<const uint2*>(src + d);
          qf[mt][ks][e] = v.x;
          qf[mt][ks][2 + e] = v.y;
        }
      }

    float o[MT][HD / 8][4];
    float m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[mt][e] = kFirstMax;
        l[mt][e] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
    }

    // ---- this key group's tiles: key0 + 32 (kg + KG i)
    const int32_t* table = a.batch.page_table + b * a.batch.table_stride;
    const int ntiles = (key1 - key0 + kTile - 1) / kTile;
    const int mine = ntiles > kg ? (ntiles - kg + KG - 1) / KG : 0;
    // page of key (lane) of tile i, or -1
    auto page_of = [&](int i) {
      const int key = key0 + kTile * (kg + KG * i) + lane;
      if (i >= mine || key >= key1) return -1;
      const int p = __ldg(table + (key >> a.pools.page_shift));
      if (p < 0 || p >= a.pools.num_pages) {
        atomicOr(a.err, kErrBadIndex);
        return -1;
      }
      return p;
    };
    auto issue = [&](int i, int pages) {
      if (i < mine) {
        const int base = key0 + kTile * (kg + KG * i);
        const uint32_t st = ring + (i % NST) * S::kStageBytes;
        constexpr int PER = kTile * CPR / (32 * RG);
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          const int idx = x * 32 * RG + gt;
          const int key = idx / CPR, chunk = idx % CPR;
          const int p = __shfl_sync(0xffffffffu, pages, key);
          const bool live = p >= 0;
          const long long slot = live ? kv_slot(a.pools, p, kvh, (base + key) & ((1 << a.pools.page_shift) - 1)) : 0;
          const long long byte = slot * RB + chunk * 16;
          cp16(st + piece_at<RB>(key, chunk), static_cast<const uint8_t*>(a.pools.k) + byte, live);
          cp16(st + kTile * RB + piece_at<RB>(key, chunk), static_cast<const uint8_t*>(a.pools.v) + byte, live);
        }
        if constexpr (FMT != NCM_KV_BF16) {
          if (rg == 0) {
            const bool live = pages >= 0;
            const long long slot = live ? kv_slot(a.pools, pages, kvh, (base + lane) & ((1 << a.pools.page_shift) - 1)) : 0;
            cp4(st + 2 * kTile * RB + 4 * lane, a.pools.k_scale + slot, live);
            cp4(st + 2 * kTile * RB + 4 * kTile + 4 * lane, a.pools.v_scale + slot, live);
          }
        }
      }
      cp_commit();
    };
    int pages = page_of(0);
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) {
      issue(i, pages);
      pages = page_of(i + 1);
    }

    for (int i = 0; i < mine; ++i) {
      cp_wait<NST - 2>();
      group_sync();  // every warp of the group has the tile, and is done with the one before it
      issue(i + NST - 1, pages);
      pages = page_of(i + NST);
      const uint32_t st = ring + (i % NST) * S::kStageBytes;
      const int base = key0 + kTile * (kg + KG * i);

      // ---- S = Q K^T
      float sc[MT][4][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][n][e] = 0.f;
#pragma unroll
      for (int j = 0; j < CPR / 4; ++j)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const uint4 w = lds128(st + piece_at<RB>(n * 8 + r, 4 * j + c));
          const uint32_t e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int x = 0; x < WPC; ++x) {
            uint32_t b0, b1;
            if constexpr (FMT == NCM_KV_BF16) {
              b0 = e[2 * x];
              b1 = e[2 * x + 1];
            } else {
              b0 = code_pair<FMT, 0, 1>(e[x]);
              b1 = code_pair<FMT, 2, 3>(e[x]);
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mma_bf16(sc[mt][n], qf[mt][j * WPC + x], b0, b1);
          }
        }

      // ---- scores in units of log2, masked where the row does not see the key
      float2 vs[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float2 f = make_float2(a.scale_log2, a.scale_log2);
        if constexpr (FMT != NCM_KV_BF16) {
          const float* scales = reinterpret_cast<const float*>(smem + (st - smem_u32(smem)) + 2 * kTile * RB);
          const float2 ks = *reinterpret_cast<const float2*>(scales + n * 8 + 2 * c);
          vs[n] = *reinterpret_cast<const float2*>(scales + kTile + n * 8 + 2 * c);
          f.x *= ks.x;
          f.y *= ks.y;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          sc[mt][n][0] *= f.x;
          sc[mt][n][1] *= f.y;
          sc[mt][n][2] *= f.x;
          sc[mt][n][3] *= f.y;
        }
      }
      const bool partly = base + kTile > min(ctx, key1);  // new tokens, or the segment's end, in this tile
      uint32_t vis[MT][2];
      if (partly) {
        const uint32_t present = first_bits(key1 - base);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i2 = node[mt][e];
            uint32_t w = 0u;
            if (i2 >= 0)
              w = present & (a.mask == nullptr
                                 ? first_bits(ctx + i2 - base + 1)
                                 : mask_window(a.mask + (s.first + static_cast<long long>(i2)) * a.mask_words, a.mask_words, base - ctx));
            vis[mt][e] = w;
            w >>= 2 * c;
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              if (!((w >> (8 * n)) & 1u)) sc[mt][n][2 * e] = -INFINITY;
              if (!((w >> (8 * n + 1)) & 1u)) sc[mt][n][2 * e + 1] = -INFINITY;
            }
          }
      }

      // ---- move the maximum only where a score passes it by more than the slack
      bool move = false;
      float top[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(sc[mt][0][2 * e], sc[mt][0][2 * e + 1]);
#pragma unroll
          for (int n = 1; n < 4; ++n) x = fmaxf(x, fmaxf(sc[mt][n][2 * e], sc[mt][n][2 * e + 1]));
          top[mt][e] = x;
          move |= x > m[mt][e] + kSlack;
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[mt][e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            x = fmaxf(x, m[mt][e]);
            const float f = ex2(m[mt][e] - x);
            m[mt][e] = x;
            l[mt][e] *= f;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
              o[mt][n][2 * e] *= f;
              o[mt][n][2 * e + 1] *= f;
            }
          }
      }

      // ---- probabilities: f32 in the sum, bf16 (with the values' scales) in the product
      uint32_t pf[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) p[e] = ex2(sc[mt][n][e] - m[mt][e >> 1]);
          l[mt][0] += p[0] + p[1];
          l[mt][1] += p[2] + p[3];
          if constexpr (FMT != NCM_KV_BF16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float z = p[e] * (e & 1 ? vs[n].y : vs[n].x);
              // (a hidden key's scale may be NaN: its row is not to hear of it)
              p[e] = partly && !((vis[mt][e >> 1] >> (8 * n + 2 * c + (e & 1))) & 1u) ? 0.f : z;
            }
          }
          pf[mt][n >> 1][(n & 1) * 2] = pack_rn(p[0], p[1]);
          pf[mt][n >> 1][(n & 1) * 2 + 1] = pack_rn(p[2], p[3]);
          if constexpr (FMT == NCM_KV_BF16) {
            sc[mt][n][0] = p[0];
            sc[mt][n][1] = p[1];
            sc[mt][n][2] = p[2];
            sc[mt][n][3] = p[3];
          }
        }

      const uint32_t vst = st + kTile * RB;
      if constexpr (FMT == NCM_KV_BF16) {
        // A new token's value row may hold a NaN or an infinity and be hidden from
        // some rows: 0 * NaN would reach them. Such rows are taken out of the tile
        // and added by the rows that see them.
        if (base + kTile > ctx) {
          bool odd = false;
#pragma unroll
          for (int x = 0; x < CPR; ++x) {
            const uint4 w = lds128(vst + lane * RB + x * 16);
            const uint32_t e[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int y = 0; y < 4; ++y) odd |= (e[y] & 0x7F80u) == 0x7F80u || (e[y] & 0x7F800000u) == 0x7F800000u;
          }
          uint32_t bad = __ballot_sync(0xffffffffu, odd);
          if (bad != 0u) {
            group_sync();
            for (uint32_t left = bad; left != 0u; left &= left - 1u) {
              const int key = __ffs(left) - 1;
              const int from = (lane & ~3) | ((key >> 1) & 3);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float p = 0.f;
#pragma unroll
                  for (int n = 0; n < 4; ++n)
                    if (n == (key >> 3)) p = (key & 1) ? sc[mt][n][2 * e + 1] : sc[mt][n][2 * e];
                  p = __shfl_sync(0xffffffffu, p, from);
                  if ((vis[mt][e] >> key) & 1u) {
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) {
                      const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + (vst - smem_u32(smem)) + piece_at<RB>(key, n) + 4 * c);
                      o[mt][n][2 * e] = fmaf(p, bf16lo(w), o[mt][n][2 * e]);
                      o[mt][n][2 * e + 1] = fmaf(p, bf16hi(w), o[mt][n][2 * e + 1]);
                    }
                  }
                }
            }
            group_sync();
            if (rg == 0 && odd)
              for (int x = 0; x < CPR; ++x) sts128(vst + lane * RB + x * 16, make_uint4(0u, 0u, 0u, 0u));
            group_sync();
          }
        }
      }

      // ---- O += P V
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int key = kk * 16 + (lane & 15);
#pragma unroll
        for (int x = 0; x < CPR / 2; ++x) {
          uint32_t w[4];
          ldmatrix_x4_trans(w, vst + piece_at<RB>(key, 2 * x + (lane >> 4)));
          if constexpr (FMT == NCM_KV_BF16) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_bf16(o[mt][2 * x], pf[mt][kk], w[0], w[1]);
              mma_bf16(o[mt][2 * x + 1], pf[mt][kk], w[2], w[3]);
            }
          } else {
            // a 16-bit element is a pair of dims: the even ones, then the odd ones
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t e0 = code_pair<FMT, 0, 2>(w[2 * y]), e1 = code_pair<FMT, 0, 2>(w[2 * y + 1]);
              const uint32_t o0 = code_pair<FMT, 1, 3>(w[2 * y]), o1 = code_pair<FMT, 1, 3>(w[2 * y + 1]);
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) {
                mma_bf16(o[mt][4 * x + 2 * y], pf[mt][kk], e0, e1);
                mma_bf16(o[mt][4 * x + 2 * y + 1], pf[mt][kk], o0, o1);
              }
            }
          }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();  // the ring's memory now carries the key groups' sums

    // ---- the key groups' sums: [KG][ROWS][m, l, values]
    constexpr int STR = HD + 4;
    float* mg = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[mt][e];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        float* row = mg + (kg * ROWS + rg * 16 * MT + mt * 16 + r + 8 * e) * STR;
        if (c == 0) {
          row[0] = m[mt][e];
          row[1] = x;
        }
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          if constexpr (FMT == NCM_KV_BF16) {
            *reinterpret_cast<float2*>(row + 4 + n * 8 + 2 * c) = make_float2(o[mt][n][2 * e], o[mt][n][2 * e + 1]);
          } else if (n % 2 == 0) {
            *reinterpret_cast<float4*>(row + 4 + (n / 2) * 16 + 4 * c) =
                make_float4(o[mt][n][2 * e], o[mt][n + 1][2 * e], o[mt][n][2 * e + 1], o[mt][n + 1][2 * e + 1]);
          }
        }
      }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == units;
    float* part = a.part + (2ll * blockIdx.x + (u0 == 0 ? 1 : 0)) * ROWS * (HD + 2);
    const int rows = min(ROWS, live_rows);
    for (int x = threadIdx.x; x < rows * (HD / 4); x += S::kThreads) {
      const int row = x / (HD / 4), d = (x % (HD / 4)) * 4;
      float mm = kFirstMax;
#pragma unroll
      for (int k = 0; k < KG; ++k) mm = fmaxf(mm, mg[(k * ROWS + row) * STR]);
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const float* src = mg + (k * ROWS + row) * STR;
        const float f = ex2(src[0] - mm);
        const float4 y = *reinterpret_cast<const float4*>(src + 4 + d);
        sum = fmaf(src[1], f, sum);
        v.x = fmaf(y.x, f, v.x);
        v.y = fmaf(y.y, f, v.y);
        v.z = fmaf(y.z, f, v.z);
        v.w = fmaf(y.w, f, v.w);
      }
      if (whole) {
        const int i = (row0 + row) / a.group, head = kvh * a.group + (row0 + row) - i * a.group;
        const long long t = s.first + static_cast<long long>(i);
        const float inv = sum == 0.f ? 0.f : __frcp_rn(sum);
        *reinterpret_cast<uint2*>(a.out + t * a.out_stride + head * HD + d) =
            sum == 0.f ? make_uint2(0u, 0u) : make_uint2(pack_bf16x2(v.x * inv, v.y * inv), pack_bf16x2(v.z * inv, v.w * inv));
        if (d == 0 && a.lse != nullptr)
          a.lse[t * a.heads + head] = sum == 0.f ? -INFINITY : (mm + log2f(sum)) * 0.69314718055994531f;
      } else {
        float* dst = part + row * (HD + 2);
        if (d == 0) *reinterpret_cast<float2*>(dst) = make_float2(mm, sum);
        *reinterpret_cast<float2*>(dst + 2 + d) = make_float2(v.x, v.y);
        *reinterpret_cast<float2*>(dst + 4 + d) = make_float2(v.z, v.w);
      }
    }
    __syncthreads();
    at += u1 - u0;
    inside += u1 - u0;
  }
}

// Adds up the partial sums of one row of one item (blockIdx.x: sequence and kv
// head, blockIdx.y: row of the sequence's rows). Four warps share the CTAs
// that worked on the item; their sums are added in warp order.
template <int HD>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeArgs a, int ROWS) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int DPL = HD / 32;
  __shared__ float sh[4][HD + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / a.pools.kv_heads, kvh = blockIdx.x - b * a.pools.kv_heads;
  const Seq s = load_seq(a, b, false);
  const int row_all = blockIdx.y;
  if (row_all >= s.n * a.group) return;
  const int tile = row_all / ROWS, row = row_all - tile * ROWS;
  auto tiles = [&](const Seq& q) { return (q.n * a.group + ROWS - 1) / ROWS; };
  const int units = units_of(a, s);
  long long before = 0, all = 0;
  for (int i = lane; i < a.batch.batch; i += 32) {
    const Seq q = load_seq(a, i, false);
    const long long u = static_cast<long long>(tiles(q)) * a.pools.kv_heads * units_of(a, q);
    all += u;
    if (i < b) before += u;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  const long long x0 = before + (static_cast<long long>(kvh) * tiles(s) + tile) * units, x1 = x0 + units - 1;
  const int c0 = static_cast<int>(((x0 + 1) * a.grid - 1) / all), c1 = static_cast<int>(((x1 + 1) * a.grid - 1) / all);
  if (c0 == c1) return;
  float mm = kFirstMax, sum = 0.f, v[DPL];
#pragma unroll
  for (int d = 0; d < DPL; ++d) v[d] = 0.f;
  auto add = [&](float m2, float l2, const float* y) {
    const float top = fmaxf(mm, m2);
    const float f = ex2(mm - top), g = ex2(m2 - top);
    sum = sum * f + l2 * g;
#pragma unroll
    for (int d = 0; d < DPL; ++d) v[d] = v[d] * f + y[d] * g;
    mm = top;
  };
  for (int c = c0 + warp; c <= c1; c += 4) {
    const float* src = a.part + ((2ll * c + (c == c0 ? 1 : 0)) * ROWS + row) * (HD + 2);
    // (CTAs of a grid larger than the number of units have none between c0 and c1)
    if (all * c / a.grid == all * (c + 1) / a.grid) continue;
    float y[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) y[d] = src[2 + lane + 32 * d];
    add(src[0], src[1], y);
  }
  if (lane == 0) {
    sh[warp][0] = mm;
    sh[warp][1] = sum;
  }
#pragma unroll
  for (int d = 0; d < DPL; ++d) sh[warp][2 + lane + 32 * d] = v[d];
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < 4; ++w) {
    float y[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) y[d] = sh[w][2 + lane + 32 * d];
    add(sh[w][0], sh[w][1], y);
  }
  const int i = row_all / a.group, head = kvh * a.group + row_all - i * a.group;
  const long long t = s.first + static_cast<long long>(i);
  const float inv = sum == 0.f ? 0.f : __frcp_rn(sum);
#pragma unroll
  for (int d = 0; d < DPL; ++d)
    a.out[t * a.out_stride + head * HD + lane + 32 * d] = sum == 0.f ? 0 : f32_to_bf16(v[d] * inv);
  if (lane == 0 && a.lse != nullptr)
    a.lse[t * a.heads + head] = sum == 0.f ? -INFINITY : (mm + log2f(sum)) * 0.69314718055994531f;
}

using TreeKernel = void (*)(const TreeArgs);
struct Variant {
  TreeKernel kernel;
  int rows, threads, smem;
};
template <int HD, int FMT, int MT, int RG, int KG>
constexpr Variant variant() {
  using S = TreeShape<HD, FMT, MT, RG, KG>;
  return Variant{tree_attention_kernel<HD, FMT, MT, RG, KG>, S::kRows, S::kThreads, S::kSmem};
}

// By the rows of one kv head: few rows take the keys four groups at a time, many
// share each tile among four row groups.
constexpr int kSizes = 4;
template <int FMT>
struct Variants {
  static constexpr Variant hd64[kSizes] = {variant<64, FMT, 1, 1, 4>(), variant<64, FMT, 2, 1, 4>(), variant<64, FMT, 2, 2, 2>(),
                                           variant<64, FMT, 2, 4, 1>()};
  static constexpr Variant hd128[kSizes] = {variant<128, FMT, 1, 1, 4>(), variant<128, FMT, 1, 2, 2>(), variant<128, FMT, 1, 4, 1>(),
                                            variant<128, FMT, 1, 4, 1>()};
};

const Variant& pick(const ncm_kv_cache_t* c, int64_t rows, int* index) {
  const bool wide = c->head_dim == 128;
  const Variant* v = c->format == NCM_KV_BF16   ? (wide ? Variants<NCM_KV_BF16>::hd128 : Variants<NCM_KV_BF16>::hd64)
                     : c->format == NCM_KV_INT8 ? (wide ? Variants<NCM_KV_INT8>::hd128 : Variants<NCM_KV_INT8>::hd64)
                                                : (wide ? Variants<NCM_KV_E4M3>::hd128 : Variants<NCM_KV_E4M3>::hd64);
  const int i = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 ? 2 : 3;
  *index = (c->format * 2 + wide) * kSizes + i;
  return v[i];
}

// Contexts this short are not split (no second kernel): one unit holds all keys.
constexpr int64_t kWholeKeys = 512;
constexpr int kUnitKeys = 128;

struct Plan {
  Variant v;
  int grid, unit_keys;
  bool merge;
  uint64_t bytes;
};

int tree_plan(ncm_ctx* ctx, const char* what, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, int32_t heads,
              int32_t max_nodes, Plan* p) {
  int rc = kv_check_cache(what, cache);
  if (rc || (rc = kv_check_batch(what, batch, true))) return rc;
  if (heads < 1 || heads % cache->kv_heads != 0 || heads / cache->kv_heads > 64)
    return ncm_fail(NCM_EINVAL, "%s: %d heads must be 1 to 64 times the %d kv heads", what, heads, cache->kv_heads);
  if (max_nodes < 1 || max_nodes > 1024) return ncm_fail(NCM_EINVAL, "%s: max_nodes %d must be 1 to 1024", what, max_nodes);
  if (static_cast<int64_t>(max_nodes) * (heads / cache->kv_heads) > 32768)
    return ncm_fail(NCM_EINVAL, "%s: %d nodes of %d heads are too many rows of one kv head", what, max_nodes, heads / cache->kv_heads);
  if (static_cast<int64_t>(batch->batch) * cache->kv_heads > INT32_MAX / 64)
    return ncm_fail(NCM_EINVAL, "%s: too many sequences", what);
  int index = 0;
  p->v = pick(cache, static_cast<int64_t>(max_nodes) * (heads / cache->kv_heads), &index);
  static std::atomic<int> resident[3 * 2 * kSizes];  // CTAs of a variant on one SM
  static DeviceFlags ready[3 * 2 * kSizes];
  if (!ready[index].test(ctx->device)) {
    int n = 0;
    NCM_CUDA_TRY(cudaFuncSetAttribute(p->v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, p->v.smem));
    NCM_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, p->v.kernel, p->v.threads, p->v.smem));
    resident[index].store(std::max(1, n));
    ready[index].set(ctx->device);
  }
  const int64_t cap = static_cast<int64_t>(batch->table_width) * cache->page_size;
  p->merge = cap > kWholeKeys;
  p->unit_keys = p->merge ? kUnitKeys : static_cast<int>(kWholeKeys);
  p->grid = ctx->num_sms * resident[index].load();
  p->bytes = static_cast<uint64_t>(2) * p->grid * p->v.rows * (cache->head_dim + 2) * sizeof(float);
  return NCM_OK;
}

}  // namespace
}  // namespace ncm

using namespace ncm;

extern "C" {

int ncm_tree_attention_workspace(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, int32_t heads,
                                 int32_t max_nodes, uint64_t* bytes) {
  DeviceGuard guard(ctx);
  if (guard.status()) return guard.status();
  if (bytes == nullptr) return ncm_fail(NCM_EINVAL, "tree_attention_workspace: null result");
  *bytes = 0;
  Plan p{};
  int rc = tree_plan(ctx, "tree_attention_workspace", cache, batch, heads, max_nodes, &p);
  if (rc) return rc;
  *bytes = p.merge ? p.bytes : 0;
  return NCM_OK;
}

int ncm_tree_attention(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, const uint16_t* q,
                       int64_t q_stride, const uint32_t* tree_mask, int32_t mask_words, int32_t heads, int32_t max_nodes,
                       float scale, uint16_t* out, int64_t out_stride, float* lse, void* workspace,
                       uint64_t workspace_bytes, ncm_stream_t stream) {
  DeviceGuard guard(ctx);
  if (guard.status()) return guard.status();
  Plan p{};
  int rc = tree_plan(ctx, "tree_attention", cache, batch, heads, max_nodes, &p);
  if (rc) return rc;
  const int64_t width = static_cast<int64_t>(heads) * cache->head_dim;
  if ((rc = kv_check_rows("tree_attention", "q", q, q_stride, batch->rows, width)) ||
      (rc = kv_check_rows("tree_attention", "out", out, out_stride, batch->rows, width)))
    return rc;
  if (!aligned_to(tree_mask, 4) || !aligned_to(lse, 4)) return ncm_fail(NCM_EINVAL, "tree_attention: misaligned buffer");
  if (tree_mask != nullptr && (mask_words < 1 || mask_words > 32))
    return ncm_fail(NCM_EINVAL, "tree_attention: mask_words %d must be 1 to 32", mask_words);
  if (batch->rows == 0 || batch->batch == 0) return NCM_OK;
  if (ranges_overlap(q, 2 * ((batch->rows - 1) * q_stride + width), out, 2 * ((batch->rows - 1) * out_stride + width)))
    return ncm_fail(NCM_EINVAL, "tree_attention: q and out overlap");
  if (p.merge && (workspace == nullptr || !aligned_to(workspace, 16) || workspace_bytes < p.bytes))
    return ncm_fail(NCM_EINVAL, "tree_attention: the workspace must hold %llu bytes, 16-byte aligned", (unsigned long long)p.bytes);
  TreeArgs a{};
  a.pools = kv_pools_of(cache);
  a.batch = kv_batch_of(batch);
  a.q = q;
  a.q_stride = q_stride;
  a.mask = tree_mask;
  a.mask_words = mask_words;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.max_nodes = max_nodes;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  a.out_stride = out_stride;
  a.lse = lse;
  a.part = static_cast<float*>(workspace);
  a.unit_keys = p.unit_keys;
  a.err = ctx->d_err;
  const int64_t most_rows = static_cast<int64_t>(max_nodes) * a.group;
  const int64_t items = static_cast<int64_t>(batch->batch) * cache->kv_heads * ceil_div(most_rows, p.v.rows);
  a.grid = p.merge ? p.grid : static_cast<int>(std::min<int64_t>(items, p.grid));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  {
    Launch _launch(ctx, KID_ATTENTION, st);
    NCM_CUDA_TRY(launch_pdl(p.v.kernel, dim3(a.grid), dim3(p.v.threads), p.v.smem, st, 1, a));
  }
  if (p.merge) {
    Launch _launch(ctx, KID_ATTENTION, st);
    auto merge = cache->head_dim == 128 ? tree_merge_kernel<128> : tree_merge_kernel<64>;
    NCM_CUDA_TRY(launch_pdl(merge, dim3(batch->batch * cache->kv_heads, static_cast<unsigned>(most_rows)), dim3(128), 0, st, 1, a,
                            p.v.rows));
  }
  return NCM_OK;
}

}  // extern "C"
