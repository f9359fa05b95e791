// What the two attention kernels over the paged cache and their merge share:
// arguments, the split of the work, masks and the last steps of a row.
#pragma once

#include "kv_cache.cuh"

namespace ncm {

constexpr float kFirstMax = -1e30f;
constexpr float kSlack = 8.f;  // scores may pass the running maximum by 2^8

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
  float* part;  // [2 * grid][ROWS][4 + HD]: m, sum of p, m', -, values
  int unit_shift;  // log2 of a unit's keys
  int begin_cost;  // what beginning an item takes, in units
  int grid;  // CTAs of the attention kernel
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

__device__ __forceinline__ uint32_t pack_rn_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four codes as two pairs of f16, exactly: bytes (0, 1) and (2, 3).
template <int FMT>
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t* lo, uint32_t* hi) {
  if constexpr (FMT == NCM_KV_INT8) {
    w ^= 0x80808080u;  // 128 + code; 0x6400 | b is 1024 + b
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(*lo) : "r"(__byte_perm(w, 0x64646464u, 0x4140)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(*hi) : "r"(__byte_perm(w, 0x64646464u, 0x4342)), "r"(0x64806480u));
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(*lo), "=r"(*hi)
        : "r"(w));
  }
}
// The same of bytes (0, 2) and (1, 3).
template <int FMT>
__device__ __forceinline__ void code_pairs_strided(uint32_t w, uint32_t* even, uint32_t* odd) {
  if constexpr (FMT == NCM_KV_INT8) {
    w ^= 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(*even) : "r"(__byte_perm(w, 0x64646464u, 0x4240)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(*odd) : "r"(__byte_perm(w, 0x64646464u, 0x4341)), "r"(0x64806480u));
  } else {
    code_pairs<FMT>(__byte_perm(w, 0u, 0x3120), even, odd);
  }
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
                   s.len > kv_capacity(a.batch, a.pools);
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
__device__ __forceinline__ int units_of(const TreeArgs& a, const Seq& s) {
  return (s.len + (1 << a.unit_shift) - 1) >> a.unit_shift;
}

// x / d for x >= 0, d > 0; in 32 bits where that does, which takes a tenth of the time.
__device__ __forceinline__ long long quotient(long long x, long long d) {
  if (((x | d) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(d);
  return x / d;
}
// The work of a sequence: every item is begin_cost places, then its units.
__device__ __forceinline__ long long places_of(const TreeArgs& a, const Seq& s, int tiles) {
  return static_cast<long long>(tiles) * a.pools.kv_heads * (a.begin_cost + units_of(a, s));
}
// How `total` places are dealt out: `ctas` CTAs (no more than there are places)
// have consecutive ones each, as evenly as whole places allow.
struct Deal {
  long long total;
  int ctas;
  __device__ __forceinline__ Deal(const TreeArgs& a, long long places)
      : total(places), ctas(static_cast<int>(min(static_cast<long long>(a.grid), places))) {}
  __device__ __forceinline__ long long first(int cta) const { return cta >= ctas ? total : quotient(total * cta, ctas); }
  __device__ __forceinline__ int owner(long long place) const { return static_cast<int>(quotient((place + 1) * ctas - 1, total)); }
};
__device__ __forceinline__ long long warp_sum(long long x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
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

// The segments of one CTA, in order: runs of consecutive units of one item
// (sequence, kv head, tile of ROWS rows). Every thread walks the same ones.
// Beginning an item costs begin_cost places, so that a CTA with many short items gets fewer keys.
template <int ROWS>
struct Walk {
  long long at, hi, inside;
  int b;
  Seq s;
  int units, u0, u1, taken;  // (taken: places of the segment)
  int kvh, row0, live_rows;  // (live_rows: rows of the item from row0 on; may be more than ROWS)
  int ctx, key0, key1;

  // Whole warps; block 0 reports sequences that do not fit.
  __device__ __forceinline__ Walk(const TreeArgs& a, int block) {
    const int lane = threadIdx.x & 31;
    auto places_at = [&](int i, bool report) {
      if (i >= a.batch.batch) return 0ll;
      const Seq q = load_seq(a, i, report);
      return places_of(a, q, tiles_of<ROWS>(a, q));
    };
    const bool report = block == 0 && threadIdx.x < 32;
    const long long mine = places_at(lane, report);  // (of the first 32 sequences, which are mostly all)
    long long total = mine;
    for (int i = lane + 32; i < a.batch.batch; i += 32) total += places_at(i, report);
    total = warp_sum(total);
    const Deal deal(a, total);
    at = deal.first(block);
    hi = deal.first(block + 1);
    inside = 0;
    taken = 0;
    b = a.batch.batch;
    if (at >= hi) return;
    // the sequence that holds place `at`
    long long x = at;
    for (int b0 = 0; b0 < a.batch.batch; b0 += 32) {
      const long long u = b0 == 0 ? mine : places_at(b0 + lane, false);
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
        inside = x - __shfl_sync(0xffffffffu, before, who);
        b = b0 + who;
        break;
      }
      x -= all;
    }
  }
  __device__ __forceinline__ bool next(const TreeArgs& a) {
    for (;;) {
      at += taken;
      inside += taken;
      taken = 0;
      if (at >= hi || b >= a.batch.batch) return false;
      s = load_seq(a, b, false);
      units = units_of(a, s);
      const int tiles = tiles_of<ROWS>(a, s), places = a.begin_cost + units;
      if (inside >= places_of(a, s, tiles)) {  // (empty sequences too)
        ++b;
        inside = 0;
        continue;
      }
      const int item = static_cast<int>(quotient(inside, places));
      const int p0 = static_cast<int>(inside - static_cast<long long>(item) * places);
      const int p1 = static_cast<int>(min(static_cast<long long>(places), p0 + (hi - at)));
      taken = p1 - p0;
      u0 = max(p0 - a.begin_cost, 0);
      u1 = max(p1 - a.begin_cost, 0);
      if (u0 == u1) continue;  // the item's units are the next CTA's
      kvh = item / tiles;
      row0 = (item - kvh * tiles) * ROWS;
      live_rows = s.n * a.group - row0;
      ctx = s.len - s.n;
      key0 = u0 << a.unit_shift;
      key1 = static_cast<int>(min(static_cast<long long>(s.len), static_cast<long long>(u1) << a.unit_shift));
      return true;
    }
  }
  __device__ __forceinline__ bool whole() const { return u0 == 0 && u1 == units; }
};

// 2^(d / 2), twice: the values' sums are brought from their maximum to the
// scores' by 2^d, which alone may pass f32's range.
__device__ __forceinline__ float half_power(float d) { return ex2(0.5f * d); }
// half_power(d) / sum; 0 for a row that saw nothing.
__device__ __forceinline__ float out_factor(float sum, float d) { return sum == 0.f ? 0.f : __fdiv_rn(half_power(d), sum); }
__device__ __forceinline__ float lse_of(float m, float sum) {
  return sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.69314718055994531f;
}

// The tcgen05 kernel (tree_attention_tc.cu): its launch, and what the plan needs of it.
struct TreeTcVariant {
  void (*kernel)(const TreeArgs);
  int rows, threads, smem;
};
TreeTcVariant tree_tc_variant(int format, int head_dim, int64_t rows);

}  // namespace ncm
