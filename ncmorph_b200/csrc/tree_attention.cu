// Attention of each sequence's new tokens over the paged cache
// (ncm_tree_attention): one decoded token, or a chain or tree of drafted ones.
//
//   out = sum_k p_k v_k / sum_k p_k,  p_k = 2^(t_k - m),  t_k = log2(e) scale q.k
//
// The query rows of one kv head (its heads / kv_heads query heads of every
// node) form tiles of up to ROWS rows; an item is (sequence, kv head, tile).
// A CTA holds KG key groups of RG warps. A key group takes every KG-th tile of
// 32 keys through a cp.async ring of its own (zero-filled behind the last
// key); each of its warps holds 8 NT query rows in registers.
//
// Products are m16n8k16 with the keys on the 16-row side, S^T = K Q^T and
// O^T = V^T P^T: a decoded token has few rows (4 for 32 query heads over 8), and
// eight of them cost half of what sixteen would. S^T's registers become
// P^T's by an 8x8 transposition in the warp (movmatrix). S sums over head_dim in any
// order, so a lane reads 16 consecutive bytes of a key and Q's fragments are
// permuted to match.
//
// Codes are used as they are: int8 and e4m3 values are exact in f16, a key's
// scale multiplies its scores, and a value's scale s enters its probability's
// exponent, p' = 2^(t + log2 s - m'), with a maximum m' of its own. P is then f16,
// which costs 2^-11 of each term, or 2^-32 of the row's largest (lifted by 2^7, the
// largest is at 2^7 or above, and f16's steps end at 2^-24). Q is bf16 and becomes
// f16 with a power of two of its row taken out: exact, but for values below 2^-17 of
// the row's largest, which are off by 2^-25 of that. A bf16 cache is multiplied in
// bf16 (its values do not fit f16's range), with P as the sum of two bf16 values, which
// costs 2^-15 of each term and a second product: rounded to one, P's error is as large as the
// output's own rounding (relative to the exact output 0.0023 instead of 0.0016 over short
// contexts, and a single key's value does not come back as it is). us of one and two values,
// eight sequences of 1 to 16 thousand tokens: 4 rows 23.7 and 23.9 at head_dim 64, 38.2 and
// 39.0 at 128; 32 rows 29.6 and 31.9, 44.3 and 49.2.
//
// A maximum is only moved when a score passes it by 2^8, so most tiles
// neither reduce over lanes nor rescale. It only takes whole values: what a row's keys
// were split into changes its probabilities by powers of two, not their 16-bit rounding.
//
// Bound: the cache's bytes with few rows (single tokens of 32 sequences of up to
// 32768 tokens, 32 query over 8 kv heads of 64, int8: 70 us, 5.6 TB/s, 0.85 of a
// copy), the issue slots of softmax and conversion with 32 rows (eight tokens of eight
// sequences, int8: 33 us, 1.6 TB/s, a quarter of a copy; every warp turns every code into
// f16 for its few rows, and 255 registers leave two CTAs an SM). A short context (4 sequences
// of 200 tokens) takes 5.7 us: one launch, and a chain of four loads.
//
// Split: items are cut into units of 128 keys, and every CTA of one wave takes
// the same number of consecutive units (beginning an item counts as three more),
// whatever the sequences' lengths are: they are known on the device only. A CTA that ends inside an item
// leaves its sums in the workspace: slot 2c for an item begun by an earlier
// CTA, slot 2c + 1 for one that goes on in the next. tree_merge_kernel adds the
// slots of such items up, in order.
#include <algorithm>

#include "tree_attention.cuh"

namespace ncm {
namespace {

constexpr int kTile = 32;  // keys of one ring stage
constexpr float kLift = 7.f;  // f16 probabilities are lifted by 2^7; with the slack they stay below 2^15

// c += A B, m16n8k16; HALF: f16 operands, otherwise bf16.
template <bool HALF>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <int HD, int FMT, int NT, int RG, int KG>
struct TreeShape {
  static constexpr int kThreads = 32 * RG * KG;
  static constexpr int kRows = 8 * NT * RG;
  static constexpr int kRowBytes = HD * (FMT == NCM_KV_BF16 ? 2 : 1);
  static constexpr int kStageBytes = 2 * kTile * kRowBytes + (FMT == NCM_KV_BF16 ? 0 : 2 * kTile * 4);
  // three stages: two tiles in flight beside the one in use
  static constexpr int kStages = 3;
  // Eight rows of 64: held to 128 registers, so that four CTAs fit an SM.
  static constexpr int kMinBlocks = NT == 1 && HD == 64 ? 4 : 1;
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

template <int HD, int FMT, int NT, int RG, int KG>
__global__ void __launch_bounds__(32 * RG * KG, TreeShape<HD, FMT, NT, RG, KG>::kMinBlocks) tree_attention_kernel(const TreeArgs a) {
  using S = TreeShape<HD, FMT, NT, RG, KG>;
  constexpr bool CODES = FMT != NCM_KV_BF16;
  constexpr int RB = S::kRowBytes, CPR = RB / 16, ROWS = S::kRows, NST = S::kStages;
  constexpr int KS = HD / 16;               // k-steps of S
  constexpr int WPC = CODES ? 4 : 2;        // k-steps in a 16-byte piece
  constexpr int DPC = CODES ? 16 : 8;       // dims in a 16-byte piece
  constexpr int DT = HD / 16;               // 16-dim tiles of O^T
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kg = warp / RG, rg = warp % RG;
  const int r = lane >> 2, c = lane & 3;
  const int gt = rg * 32 + lane;  // thread of the key group
  const uint32_t ring = smem_u32(smem) + kg * NST * S::kStageBytes;
  pdl_wait();

  Walk<ROWS> w(a, blockIdx.x);
  auto group_sync = [&] {
    if constexpr (RG == 1)
      __syncwarp();
    else
      asm volatile("bar.sync %0, %1;" ::"r"(1 + kg), "n"(32 * RG) : "memory");
  };

  while (w.next(a)) {
    const Seq s = w.s;
    const int kvh = w.kvh, row0 = w.row0, live_rows = w.live_rows, ctx = w.ctx, key0 = w.key0, key1 = w.key1;

    // ---- this key group's tiles: key0 + 32 (kg + KG i)
    const int32_t* table = a.batch.page_table + w.b * a.batch.table_stride;
    const int ntiles = (key1 - key0 + kTile - 1) / kTile;
    const int mine = ntiles > kg ? (ntiles - kg + KG - 1) / KG : 0;
    const int page_mask = (1 << a.pools.page_shift) - 1;
    // page of key (lane) of tile i (asked for one tile ahead of its use); -1 behind the last key
    auto page_of = [&](int i) {
      const int key = key0 + kTile * (kg + KG * i) + lane;
      return i < mine && key < key1 ? __ldg(table + (key >> a.pools.page_shift)) : -1;
    };
    auto issue = [&](int i, int pages) {
      if (i < mine) {
        if (pages < 0 || pages >= a.pools.num_pages) {
          if (key0 + kTile * (kg + KG * i) + lane < key1) atomicOr(a.err, kErrBadIndex);
          pages = -1;
        }
        const int base = key0 + kTile * (kg + KG * i);
        const uint32_t st = ring + (i % NST) * S::kStageBytes;
        constexpr int PER = kTile * CPR / (32 * RG);
        const int off = (base + lane) & page_mask;
        const long long slot = pages >= 0 ? kv_slot(a.pools, pages, kvh, off) : 0;
        if (a.pools.page_shift >= 5) {  // the tile is one run of its page
          const long long first = __shfl_sync(0xffffffffu, slot, 0) * RB + gt * 16;
          const int live = __popc(__ballot_sync(0xffffffffu, pages >= 0));  // its first keys
          const uint8_t* ks = static_cast<const uint8_t*>(a.pools.k) + first;
          const uint8_t* vs = static_cast<const uint8_t*>(a.pools.v) + first;
#pragma unroll
          for (int x = 0; x < PER; ++x) {
            const int idx = x * 32 * RG + gt;
            const int key = idx / CPR;
            const uint32_t to = st + piece_at<RB>(key, idx % CPR);
            cp16(to, ks + (key < live ? x * 512 * RG : 0), key < live);
            cp16(to + kTile * RB, vs + (key < live ? x * 512 * RG : 0), key < live);
          }
        } else {
#pragma unroll
          for (int x = 0; x < PER; ++x) {
            const int idx = x * 32 * RG + gt;
            const int key = idx / CPR, chunk = idx % CPR;
            const bool live = __shfl_sync(0xffffffffu, pages, key) >= 0;
            const long long byte = __shfl_sync(0xffffffffu, slot, key) * RB + chunk * 16;
            const uint32_t to = st + piece_at<RB>(key, chunk);
            cp16(to, static_cast<const uint8_t*>(a.pools.k) + byte, live);
            cp16(to + kTile * RB, static_cast<const uint8_t*>(a.pools.v) + byte, live);
          }
        }
        if constexpr (CODES) {
          if (rg == 0) {
            cp4(st + 2 * kTile * RB + 4 * lane, a.pools.k_scale + slot, pages >= 0);
            cp4(st + 2 * kTile * RB + 4 * kTile + 4 * lane, a.pools.v_scale + slot, pages >= 0);
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

    // ---- this warp's query rows (row r of each n-tile), in fragment order
    uint32_t qf[NT][KS][2];
    float row_scale[NT][2];  // of rows 2c and 2c + 1: what their scores are multiplied by
    int node[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int base = row0 + rg * 8 * NT + nt * 8;
      const int row = base + r;
      const bool live = row < row0 + live_rows;
      const int i = live ? row / a.group : 0;
      const int head = kvh * a.group + (live ? row - i * a.group : 0);
      const uint16_t* src = a.q + (s.first + static_cast<long long>(i)) * a.q_stride + head * HD;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = ((ks / WPC) * 4 + c) * DPC + (ks % WPC) * 4;
        uint2 v = make_uint2(0u, 0u);
        if (live) v = *reinterpret_cast<const uint2*>(src + d);
        qf[nt][ks][0] = v.x;
        qf[nt][ks][1] = v.y;
      }
      float up = 1.f;  // (row r's own)
      if constexpr (CODES) {
        uint32_t top = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e) top = max(top, max(qf[nt][ks][e] & 0x7FFFu, (qf[nt][ks][e] >> 16) & 0x7FFFu));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest becomes 1 to 2 (2 to 4 at the top of bf16's range)
        const uint32_t ex = top >> 7, f = min(max(254 - static_cast<int>(ex), 1), 253);
        const float down = __uint_as_float(f << 23);
        up = __uint_as_float((254u - f) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            qf[nt][ks][e] = pack_rn_f16x2(bf16lo(qf[nt][ks][e]) * down, bf16hi(qf[nt][ks][e]) * down);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row_scale[nt][e] = a.scale_log2 * __shfl_sync(0xffffffffu, up, (2 * c + e) * 4);
        const int mine_row = base + 2 * c + e;
        node[nt][e] = mine_row < row0 + live_rows ? mine_row / a.group : -1;
      }
    }

    float o[DT][NT][4];           // dims r and r + 8 (codes: 2 r and 2 r + 1) of each 16, rows 2c and 2c + 1
    float m[NT][2], mv[NT][2], l[NT][2];  // maxima of the scores, and with the values' scales; sums
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nt][e] = mv[nt][e] = kFirstMax;
        l[nt][e] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][nt][e] = 0.f;
    }

    for (int i = 0; i < mine; ++i) {
      cp_wait<NST - 2>();
      group_sync();  // every warp of the group has the tile, and is done with the one before it
      issue(i + NST - 1, pages);
      pages = page_of(i + NST);
      const uint32_t off = (ring - smem_u32(smem)) + (i % NST) * S::kStageBytes;
      const uint32_t st = smem_u32(smem) + off;
      const int base = key0 + kTile * (kg + KG * i);

      // ---- S^T = K Q^T: sc[mt][nt]: keys 16 mt + r (0, 1) and + 8 (2, 3), rows 2c (0, 2) and 2c + 1 (1, 3)
      float sc[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[mt][nt][e] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int j = 0; j < CPR / 4; ++j) {
          const uint4 x = lds128(st + piece_at<RB>(mt * 16 + r, 4 * j + c));
          const uint4 y = lds128(st + piece_at<RB>(mt * 16 + 8 + r, 4 * j + c));
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int w = 0; w < WPC; ++w) {
            uint32_t f[4];
            if constexpr (CODES) {
              code_pairs<FMT>(xs[w], &f[0], &f[2]);
              code_pairs<FMT>(ys[w], &f[1], &f[3]);
            } else {
              f[0] = xs[2 * w];
              f[1] = ys[2 * w];
              f[2] = xs[2 * w + 1];
              f[3] = ys[2 * w + 1];
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16<CODES>(sc[mt][nt], f, qf[nt][j * WPC + w][0], qf[nt][j * WPC + w][1]);
          }
        }

      // ---- scores in units of log2, masked where the row does not see the key
      float vlog[2][2];  // log2 of the values' scales of keys 16 mt + 8 h + r
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float ks = 1.f;
          if constexpr (CODES) {
            const float* scales = reinterpret_cast<const float*>(smem + off + 2 * kTile * RB) + mt * 16 + h * 8 + r;
            ks = scales[0];
            vlog[mt][h] = lg2(scales[kTile]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float t = sc[mt][nt][2 * h + e] * row_scale[nt][e];
              if constexpr (CODES) t *= ks;
              sc[mt][nt][2 * h + e] = t;
            }
        }
      const bool partly = base + kTile > min(ctx, key1);  // new tokens, or the segment's end, in this tile
      uint32_t vis[NT][2];
      if (partly) {
        const uint32_t present = first_bits(key1 - base);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i2 = node[nt][e];
            uint32_t w = 0u;
            if (i2 >= 0)
              w = present & (a.mask == nullptr
                                 ? first_bits(ctx + i2 - base + 1)
                                 : mask_window(a.mask + (s.first + static_cast<long long>(i2)) * a.mask_words, a.mask_words, base - ctx));
            vis[nt][e] = w;
            w >>= r;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (!((w >> (16 * mt + 8 * h)) & 1u)) sc[mt][nt][2 * h + e] = -INFINITY;
          }
      }

      // ---- move a maximum only where a score passes it by more than the slack
      bool move = false;
      float top[NT][2], topv[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][2 + e]), fmaxf(sc[1][nt][e], sc[1][nt][2 + e]));
          move |= top[nt][e] > m[nt][e] + kSlack;
          if constexpr (CODES) {
            topv[nt][e] = fmaxf(fmaxf(sc[0][nt][e] + vlog[0][0], sc[0][nt][2 + e] + vlog[0][1]),
                                fmaxf(sc[1][nt][e] + vlog[1][0], sc[1][nt][2 + e] + vlog[1][1]));
            move |= topv[nt][e] > mv[nt][e] + (kSlack + kLift);
          }
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = top[nt][e];
#pragma unroll
            for (int z = 4; z < 32; z <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, z));
            x = fmaxf(ceilf(x), m[nt][e]);
            float f = ex2(m[nt][e] - x);
            m[nt][e] = x;
            l[nt][e] *= f;
            if constexpr (CODES) {
              x = topv[nt][e];
#pragma unroll
              for (int z = 4; z < 32; z <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, z));
              x = fmaxf(floorf(x - kLift), mv[nt][e]);
              f = ex2(mv[nt][e] - x);
              mv[nt][e] = x;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              o[d][nt][e] *= f;
              o[d][nt][2 + e] *= f;
            }
          }
      }

      // ---- probabilities: f32 in the sum, f16 with the values' scales in the product over codes
      uint32_t pf[2][NT][2];  // P^T: keys 16 mt + 2c, + 1 (0) and + 8 (1) of row r
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float p[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float t = sc[mt][nt][2 * h + e];
              p[e] = ex2(t - m[nt][e]);
              l[nt][e] += p[e];
              if constexpr (CODES) {
                p[e] = ex2(t + vlog[mt][h] - mv[nt][e]);
                // (a hidden key's scale may be NaN: its row is not to hear of it)
                if (partly && !((vis[nt][e] >> (16 * mt + 8 * h + r)) & 1u)) p[e] = 0.f;
              } else {
                sc[mt][nt][2 * h + e] = p[e];
              }
            }
            if constexpr (CODES) pf[mt][nt][h] = transpose8x8(pack_rn_f16x2(p[0], p[1]));
          }

      const uint32_t vst = st + kTile * RB;
      if constexpr (!CODES) {
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
          const uint32_t bad = __ballot_sync(0xffffffffu, odd);
          if (bad != 0u) {
            group_sync();
            for (uint32_t left = bad; left != 0u; left &= left - 1u) {
              const int key = __ffs(left) - 1;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float p = 0.f;
#pragma unroll
                  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                      if (key >> 3 == 2 * mt + h) p = sc[mt][nt][2 * h + e];
                  p = __shfl_sync(0xffffffffu, p, (key & 7) * 4 + c);
                  if ((vis[nt][e] >> key) & 1u) {
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                      for (int h = 0; h < 2; ++h) {
                        const uint16_t v = *reinterpret_cast<const uint16_t*>(smem + off + kTile * RB + piece_at<RB>(key, 2 * d + h) + 2 * r);
                        o[d][nt][2 * h + e] = fmaf(p, bf16_to_f32(v), o[d][nt][2 * h + e]);
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

      // ---- O^T += V^T P^T
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        // P is cut off behind bf16's bits, and what that left is the second value. It is above 0
        // (2^-20 of P are added), so that a value that is infinite stays so: both parts
        // of its product have its sign, and neither is 0 times it.
        constexpr float kAbove1 = 1.f + 0x1p-20f;
        uint32_t rest[NT][2];
        if constexpr (!CODES) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float p0 = sc[kk][nt][2 * h], p1 = sc[kk][nt][2 * h + 1];
              const uint32_t top = __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
              pf[kk][nt][h] = transpose8x8(top);
              rest[nt][h] = transpose8x8(pack_rn_bf16x2(fmaf(p0, kAbove1, -bf16lo(top)), fmaf(p1, kAbove1, -bf16hi(top))));
            }
        }
#pragma unroll
        for (int x = 0; x < CPR / 2; ++x) {
          uint32_t w[4];
          if constexpr (CODES) {  // 16-bit elements are pairs of dims: the even ones become rows r, the odd ones rows r + 8
            ldmatrix_x4_trans(w, vst + piece_at<RB>(kk * 16 + (lane & 15), 2 * x + (lane >> 4)));
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t f[4];
              code_pairs_strided<FMT>(w[2 * y], &f[0], &f[1]);
              code_pairs_strided<FMT>(w[2 * y + 1], &f[2], &f[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16<true>(o[2 * x + y][nt], f, pf[kk][nt][0], pf[kk][nt][1]);
            }
          } else {
            ldmatrix_x4_trans(w, vst + piece_at<RB>(kk * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * x + ((lane >> 3) & 1)));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16<false>(o[x][nt], w, pf[kk][nt][0], pf[kk][nt][1]);
              mma16<false>(o[x][nt], w, rest[nt][0], rest[nt][1]);
            }
          }
        }
      }
    }
    cp_wait<0>();
    __syncthreads();  // the ring's memory now carries the key groups' sums

    // ---- the key groups' sums: [KG][ROWS][m, l, m', -, values]
    constexpr int STR = HD + 4;
    float* mg = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[nt][e];
#pragma unroll
        for (int z = 4; z < 32; z <<= 1) x += __shfl_xor_sync(0xffffffffu, x, z);
        float* row = mg + (kg * ROWS + rg * 8 * NT + nt * 8 + 2 * c + e) * STR;
        if (r == 0) *reinterpret_cast<float4*>(row) = make_float4(m[nt][e], x, CODES ? mv[nt][e] : m[nt][e], 0.f);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          if constexpr (CODES) {
            *reinterpret_cast<float2*>(row + 4 + 16 * d + 2 * r) = make_float2(o[d][nt][e], o[d][nt][2 + e]);
          } else {
            row[4 + 16 * d + r] = o[d][nt][e];
            row[4 + 16 * d + 8 + r] = o[d][nt][2 + e];
          }
        }
      }
    __syncthreads();
    const bool whole = w.whole();
    float* part = a.part + (2ll * blockIdx.x + (w.u0 == 0 ? 1 : 0)) * ROWS * STR;
    const int rows = min(ROWS, live_rows);
    for (int x = threadIdx.x; x < rows * (HD / 4); x += S::kThreads) {
      const int row = x / (HD / 4), d = (x % (HD / 4)) * 4;
      float4 top = *reinterpret_cast<const float4*>(mg + row * STR);
#pragma unroll
      for (int k = 1; k < KG; ++k) {
        const float* src = mg + (k * ROWS + row) * STR;
        top.x = fmaxf(top.x, src[0]);
        top.z = fmaxf(top.z, src[2]);
      }
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const float* src = mg + (k * ROWS + row) * STR;
        const float f = ex2(src[2] - top.z);
        const float4 y = *reinterpret_cast<const float4*>(src + 4 + d);
        sum = fmaf(src[1], ex2(src[0] - top.x), sum);
        v.x = fmaf(y.x, f, v.x);
        v.y = fmaf(y.y, f, v.y);
        v.z = fmaf(y.z, f, v.z);
        v.w = fmaf(y.w, f, v.w);
      }
      if (whole) {
        const int i = (row0 + row) / a.group, head = kvh * a.group + (row0 + row) - i * a.group;
        const long long t = s.first + static_cast<long long>(i);
        const float f = out_factor(sum, top.z - top.x);
        const float g = half_power(top.z - top.x);
        *reinterpret_cast<uint2*>(a.out + t * a.out_stride + head * HD + d) =
            make_uint2(pack_rn_bf16x2(v.x * f * g, v.y * f * g), pack_rn_bf16x2(v.z * f * g, v.w * f * g));
        if (d == 0 && a.lse != nullptr) a.lse[t * a.heads + head] = lse_of(top.x, sum);
      } else {
        float* dst = part + row * STR;
        if (d == 0) *reinterpret_cast<float4*>(dst) = make_float4(top.x, sum, top.z, 0.f);
        *reinterpret_cast<float4*>(dst + 4 + d) = v;
      }
    }
    __syncthreads();
  }
}

// Adds up the partial sums of a row of an item (blockIdx.x: sequence and kv
// head, blockIdx.y: 4 / WPR rows of the sequence's rows), in an order that the
// split alone decides. WPR warps share a row: all four of the block where there are few
// rows (kManyRows), otherwise one. Each row's warps look all sequences up for their places, which
// grows with rows x sequences: 4 of the 14 us of 32 sequences of up to 1600 keys, 265 of
// 600 us of 2048. What the caller
// gave is read before the wait: the attention kernel does not let this one start
// ahead of its own end, and the kernels in front of both are done by then.
constexpr int kMaxParts = 2048;  // CTAs of the attention kernel at most

template <int HD, int WPR>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeArgs a, int ROWS) {
  constexpr int STR = HD + 4, LPP = HD / 4, GROUPS = 32 * WPR / LPP;  // lanes of a part, parts at a time
  __shared__ float red[4][3];
  __shared__ float4 vals[WPR == 4 ? GROUPS : 1][LPP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tid = threadIdx.x % (32 * WPR);  // of the row's threads
  const int b = blockIdx.x / a.pools.kv_heads, kvh = blockIdx.x - b * a.pools.kv_heads;
  const Seq s = load_seq(a, b, false);
  const int row_all = blockIdx.y * (4 / WPR) + (WPR == 1 ? warp : 0);
  const int tile = row_all / ROWS, row = row_all - tile * ROWS;
  auto tiles = [&](const Seq& q) { return (q.n * a.group + ROWS - 1) / ROWS; };
  const int units = units_of(a, s);
  long long before = 0, total = 0;
  for (int i = lane; i < a.batch.batch; i += 32) {
    const Seq q = load_seq(a, i, false);
    const long long u = places_of(a, q, tiles(q));
    total += u;
    if (i < b) before += u;
  }
  before = warp_sum(before);
  total = warp_sum(total);
  const long long x0 = before + (static_cast<long long>(kvh) * tiles(s) + tile) * (a.begin_cost + units) + a.begin_cost;
  const Deal deal(a, total);
  const bool exists = row_all < s.n * a.group;
  const int c0 = exists ? deal.owner(x0) : 0, c1 = exists ? deal.owner(x0 + units - 1) : 0;
  pdl_wait();
  pdl_launch_dependents();
  if (c0 == c1) return;  // no such row, or one CTA had the whole item and wrote its rows
  const int n = c1 - c0 + 1;
  const float* first = a.part + row * STR;
  auto part_of = [&](int k) { return first + (2ll * (c0 + k) + (k == 0 ? 1 : 0)) * ROWS * STR; };
  // ---- maxima, then the sum with the parts' weights
  float mm = kFirstMax, mv = kFirstMax;
  for (int k = tid; k < n; k += 32 * WPR) {
    const float4 h = *reinterpret_cast<const float4*>(part_of(k));
    mm = fmaxf(mm, h.x);
    mv = fmaxf(mv, h.z);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
    mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, o));
  }
  if constexpr (WPR == 4) {
    if (lane == 0) {
      red[warp][0] = mm;
      red[warp][1] = mv;
    }
    __syncthreads();
    mm = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
    mv = fmaxf(fmaxf(red[0][1], red[1][1]), fmaxf(red[2][1], red[3][1]));
  }
  float sum = 0.f;
  for (int k = tid; k < n; k += 32 * WPR) {
    const float4 h = *reinterpret_cast<const float4*>(part_of(k));
    sum = fmaf(h.y, ex2(h.x - mm), sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if constexpr (WPR == 4) {
    if (lane == 0) red[warp][2] = sum;
    __syncthreads();
    sum = (red[0][2] + red[1][2]) + (red[2][2] + red[3][2]);
  }
  // ---- values, four parts of a group of lanes in flight
  const int g = tid / LPP, d = tid % LPP;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = g; k0 < n; k0 += 4 * GROUPS) {
    float4 y[4];
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + i * GROUPS;
      w[i] = kFirstMax;
      y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k < n) {
        const float* p = part_of(k);
        w[i] = p[2];
        y[i] = *reinterpret_cast<const float4*>(p + 4 + 4 * d);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = ex2(w[i] - mv);
      v.x = fmaf(y[i].x, f, v.x);
      v.y = fmaf(y[i].y, f, v.y);
      v.z = fmaf(y[i].z, f, v.z);
      v.w = fmaf(y[i].w, f, v.w);
    }
  }
  if constexpr (WPR == 4) {
    vals[g][d] = v;
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int k = 1; k < GROUPS; ++k) {
      const float4 y = vals[k][d];
      v.x += y.x;
      v.y += y.y;
      v.z += y.z;
      v.w += y.w;
    }
  } else if constexpr (GROUPS == 2) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, 16);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
    v.z += __shfl_xor_sync(0xffffffffu, v.z, 16);
    v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
    if (g != 0) return;
  }
  const int i = row_all / a.group, head = kvh * a.group + row_all - i * a.group;
  const long long t = s.first + static_cast<long long>(i);
  const float f = out_factor(sum, mv - mm), h = half_power(mv - mm);
  *reinterpret_cast<uint2*>(a.out + t * a.out_stride + head * HD + 4 * d) =
      make_uint2(pack_rn_bf16x2(v.x * f * h, v.y * f * h), pack_rn_bf16x2(v.z * f * h, v.w * f * h));
  if (d == 0 && a.lse != nullptr) a.lse[t * a.heads + head] = lse_of(mm, sum);
}

using Variant = TreeTcVariant;
template <int HD, int FMT, int NT, int RG, int KG>
constexpr Variant variant() {
  using S = TreeShape<HD, FMT, NT, RG, KG>;
  return Variant{tree_attention_kernel<HD, FMT, NT, RG, KG>, S::kRows, S::kThreads, S::kSmem};
}

// By the rows of one kv head: 8, 16 or 32 rows a tile. Few rows take the
// keys four groups at a time, more share each tile among row groups.
constexpr int kSizes = 3;
template <int FMT>
struct Variants {
  static constexpr Variant hd64[kSizes] = {variant<64, FMT, 1, 1, 4>(), variant<64, FMT, 2, 1, 4>(), variant<64, FMT, 4, 1, 4>()};
  static constexpr Variant hd128[kSizes] = {variant<128, FMT, 1, 1, 4>(), variant<128, FMT, 2, 1, 4>(), variant<128, FMT, 2, 2, 2>()};
};

// Rows of one kv head that stay with the mma.sync kernel. More go to the tcgen05
// kernel, whose tiles have 128 rows. us of both, mma.sync / tcgen05 (eight
// sequences of 1 to 16 thousand tokens, 8 kv heads): 32 rows, bf16: 32 / 40 at
// head_dim 64, 49 / 63 at 128, int8: 33 / 44 and 48 / 65; 48 rows (bf16 with P as one
// value): 40 / 41, 67 / 64, 48 / 45 and 78 / 69; 64 rows: 41 / 42, 68 / 65, 49 / 45 and 79 / 70.
constexpr int64_t kFewRows = 32;
Variant pick(const ncm_kv_cache_t* c, int64_t rows, int* index) {
  const bool wide = c->head_dim == 128;
  if (rows > kFewRows) {
    *index = 3 * 2 * kSizes + (c->format * 2 + wide) * 2 + (rows > 128);
    return tree_tc_variant(c->format, c->head_dim, rows);
  }
  const Variant* v = c->format == NCM_KV_BF16   ? (wide ? Variants<NCM_KV_BF16>::hd128 : Variants<NCM_KV_BF16>::hd64)
                     : c->format == NCM_KV_INT8 ? (wide ? Variants<NCM_KV_INT8>::hd128 : Variants<NCM_KV_INT8>::hd64)
                                                : (wide ? Variants<NCM_KV_E4M3>::hd128 : Variants<NCM_KV_E4M3>::hd64);
  const int i = rows <= 8 ? 0 : rows <= 16 ? 1 : 2;
  *index = (c->format * 2 + wide) * kSizes + i;
  return v[i];
}

// Contexts this short are not split (no second kernel): one unit holds all keys.
constexpr int kWholeShift = 9;
constexpr int kUnitShift = 7;
// What beginning an item costs (query rows, the first keys' way, the sums' way out), in
// units. us at 0, 2, 3 and 4, eight to 32 sequences of 1 to 16 thousand tokens: one token,
// bf16, head_dim 64: 39.1, 37.5, 36.8, 37.0; eight, int8: 43.1, 37.8, 33.7, 33.0; 26
// (tcgen05), e4m3, head_dim 128: 73, 58.0, 55.8, 55.9; one long sequence: no difference.
constexpr int kBeginCost = 3;

// Rows of the merge an SM, from which one warp adds up a row; fewer are shared by four
// warps each. us of four / one: 256 rows of 9 parts: 19.9 / 20.6, 512 rows of 55:
// 45.1 / 45.3 (head_dim 128: 34.4 / 35.3), 2048 rows of 18: 76.2 / 72.9, 4096 of 9: 146 / 139.
constexpr int kManyRows = 6;

struct Plan {
  Variant v;
  int grid, unit_shift;
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
  static DeviceNumbers resident[3 * 2 * (kSizes + 2)];  // CTAs of a variant on one SM of a device
  int on_sm = resident[index].get(ctx->device);
  if (on_sm == 0) {
    NCM_CUDA_TRY(cudaFuncSetAttribute(p->v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, p->v.smem));
    NCM_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&on_sm, p->v.kernel, p->v.threads, p->v.smem));
    on_sm = std::max(1, on_sm);
    resident[index].set(ctx->device, on_sm);
  }
  const int64_t cap = std::min<int64_t>(static_cast<int64_t>(batch->table_width) * cache->page_size, 1 << 30);
  p->merge = cap > 1 << kWholeShift;
  p->unit_shift = p->merge ? kUnitShift : kWholeShift;
  const int64_t tiles = ceil_div(static_cast<int64_t>(max_nodes) * (heads / cache->kv_heads), p->v.rows);
  // (the kernels multiply the number of units by that of the CTAs)
  if (batch->batch * cache->kv_heads * tiles * (kBeginCost + ceil_div(cap, 1 << p->unit_shift)) > INT64_MAX / (2 * kMaxParts))
    return ncm_fail(NCM_EINVAL, "%s: too many keys", what);
  p->grid = std::min(kMaxParts, ctx->num_sms * on_sm);
  p->bytes = static_cast<uint64_t>(2) * p->grid * p->v.rows * (cache->head_dim + 4) * sizeof(float);
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
  a.unit_shift = p.unit_shift;
  a.begin_cost = kBeginCost;
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
    const bool wide = cache->head_dim == 128, few = static_cast<int64_t>(batch->batch) * cache->kv_heads * most_rows < kManyRows * ctx->num_sms;
    auto merge = few ? (wide ? tree_merge_kernel<128, 4> : tree_merge_kernel<64, 4>)
                     : (wide ? tree_merge_kernel<128, 1> : tree_merge_kernel<64, 1>);
    NCM_CUDA_TRY(launch_pdl(merge, dim3(batch->batch * cache->kv_heads, ceil_div(most_rows, few ? 1 : 4)), dim3(128), 0, st, 1, a, p.v.rows));
  }
  return NCM_OK;
}

}  // extern "C"
