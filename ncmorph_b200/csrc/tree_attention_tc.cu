// Attention of many drafted tokens over the paged cache: the same operator, split
// and partial sums as tree_attention.cu, for items whose query rows fill more of a
// 128-row tensor-core tile (rows: nodes x the query heads of one kv head). Per key
// tile of 64:
//   S = Q K^T    tcgen05.mma M=128 N=64 K=head_dim, f32 in tensor memory (two buffers)
//   softmax      one thread per row; P (bf16) into a 128-byte-swizzled tile
//   O += P V     tcgen05.mma M=128 N=head_dim K=64, accumulated in tensor memory
// Two groups of four softmax warps work side by side: with up to 128 rows they
// take every other key tile and add their sums up at the end, with more
// (head_dim 64) each has 128 rows of its own. One warp per group issues its
// products, in whatever order their operands come; the others load. Every key
// and value is fetched and, for int8 and e4m3, turned into bf16 (exactly) once per CTA,
// whatever the number of rows; in the mma.sync kernel each 8 to 32 rows do that again.
// A key's scale multiplies its scores, a value's scale its probability. V is
// taken as it lies in the cache, head_dim contiguous: the second product's B
// operand is MN-major.
//
// Bound: the exponentials (16 a clock and SM: 64 keys of 128 rows take 512 clocks, the
// two products 256 at head_dim 64 and 512 at 128). Two trees of 64 tokens over up to 131072
// tokens, bf16, head_dim 64 (256 rows): 136 us, 535 TFLOP/s; the special-function unit
// is busy half of the kernel's time, and a group's 64 keys take 2000 clocks, 1024 of
// them exponentials of both groups. Trees of 26 tokens of eight sequences of up to 8191 tokens, e4m3,
// head_dim 128 (104 rows): 48 us, 179 TFLOP/s; a CTA has about ten tiles of each group there,
// and its start (a chain of lookups and the first keys: 10000 clocks), the sums' way out and
// the merge are half of the time. The 96 registers of 576 threads spill 36 to 76 bytes, the 128 of
// 448 threads 16 over codes, none over bf16. The maximum moves only past 2^8 (kSlack), as in the other
// kernel; then O is rescaled in tensor memory.
//
// A value row of a new token that holds a NaN or an infinity and is hidden from some rows
// must not reach them as 0 * NaN: the loaders put zeros in the place of such values, and
// rows that see them add them at the end.
#include "tree_attention.cuh"

namespace ncm {
namespace {

constexpr int kLoadWarps = 4;  // of a group
constexpr int kLoadThreads = 32 * kLoadWarps;

struct TcBars {
  uint64_t q_full;
  uint64_t k_full[8], k_empty[8], v_full[8], v_empty[8];
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2];  // [group][buffer]
  uint64_t sums_full[4], taken[4];  // [pair of the groups' warps] their sums are there; both have read both groups' values
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort_flag;
  int odd_values;  // a loader met a value that is not finite in a tile of new tokens
};
constexpr int kBarBytes = 512;
static_assert(sizeof(TcBars) <= kBarBytes, "barriers");

// SPLITQ: the groups have 128 rows each; otherwise the same 128 rows and every other tile.
template <int HD, int FMT, bool SPLITQ>
struct TcShape {
  static_assert(!SPLITQ || HD == 64, "256 rows fit with head_dim 64 only");
  static constexpr bool kCodes = FMT != NCM_KV_BF16;
  static constexpr int kQTiles = SPLITQ ? 2 : 1;
  static constexpr int kRows = 128 * kQTiles;
  // Two groups of loaders take every other tile, so that one's waits and conversion run
  // beside the other's. A tile that 256 rows share lasts long enough for one group, which
  // leaves 128 registers a thread (int8, eight sequences of 64 tokens: 80.3 us with two
  // groups, 77.5 with one; 128 rows, bf16: 45.5 and 51.9).
  static constexpr int kLoadGroups = SPLITQ ? 1 : 2;
  static constexpr int kThreads = 32 * (8 + 2 + kLoadGroups * kLoadWarps);
  static constexpr int kRowBytes = HD * (kCodes ? 1 : 2);
  static constexpr int kBK = 64;  // keys of a tile
  // Tiles in bf16, and for codes the raw tiles in flight in front of them.
  static constexpr int kStages = HD == 64 ? (kCodes ? 4 : 8) : (kCodes ? 2 : 4);
  static constexpr int kRaw = kCodes ? 4 : 0;
  // Buffers of P, of 128 rows x kBK keys (one where shared memory is full).
  static constexpr int kPBufs = kCodes && HD == 128 ? 1 : 2;
  static constexpr int kPBytes = 256 * kBK;
  // tiles that a group of loaders has asked for before it waits for the first of them
  static constexpr int kAhead = kLoadGroups == 1 ? 4 : 2;
  // (a stage's uses all belong to one group of loaders, and to one of softmax warps
  // where those take every other tile: each waits for its own earlier use)
  static_assert(kStages % 2 == 0, "stages per group");
  // Slots of the scales: a K stage is free again when its S is issued, up to two tiles of
  // its group ahead of the softmax that still reads an earlier tile's scales.
  static constexpr int kScaleSlots = kStages + 8;
  static constexpr int kBlocks = HD / 64;  // 64-dim columns of a tile
  static constexpr int kQ = 0;
  static constexpr int kP = kQ + kQTiles * kBlocks * 16384;  // [group][buffer]
  static constexpr int kK = kP + 2 * kPBufs * kPBytes;
  static constexpr int kBlock = 128 * kBK;  // bytes of 64 dims of a K or V tile
  static constexpr int kV = kK + kStages * kBlocks * kBlock;
  static constexpr int kRawAt = kV + kStages * kBlocks * kBlock;
  static constexpr int kScale = kRawAt + kRaw * 2 * kBK * kRowBytes;  // [slot][K (times log2(e) scale), V][kBK] f32
  static constexpr int kRawScale = kScale + (kCodes ? kScaleSlots * 2 * kBK * 4 : 0);  // [raw][K, V][kBK] f32
  static constexpr int kBars = kRawScale + kRaw * 2 * kBK * 4;
  static constexpr int kSums = kBars + kBarBytes;  // !SPLITQ: the groups' maxima and sums, [group][128]
  static constexpr int kSmem = kSums + (SPLITQ ? 0 : 2 * 128 * 8);
  static constexpr uint32_t kTmemCols = 512;  // S: 2 x 2 x 64, O: 2 x head_dim
  static_assert(kSmem <= 232448, "shared memory of the tcgen05 attention");
};

// Instruction descriptor: bf16 operands, f32 sums, M = 128; B MN-major where `mn`.
__device__ constexpr uint32_t tc_idesc(int n, bool mn) { return idesc_bf16_f32(128, n) | (mn ? 1u << 16 : 0u); }

// Descriptor of an MN-major bf16 tile with 128-byte swizzling: rows (the
// contracted index) of 64 elements, 8-row groups 1024 bytes apart, further
// 64-element columns `column` bytes apart.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr, uint32_t column) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | static_cast<uint64_t>(column >> 4) << 16 |
         static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}

// Bytes I and J of w as two bf16 values, exactly. int8: 128 + (low seven bits) minus
// 128 or 256, by the sign bit. e4m3: the code's exponent and mantissa moved into
// bf16's fields are the value times 2^-120 (subnormal codes included).
template <int FMT>
__device__ __forceinline__ uint32_t code_pair_bf16(uint32_t w, uint32_t hi) {
  uint32_t r;
  if constexpr (FMT == NCM_KV_INT8) {
    const uint32_t x = __byte_perm(w, 0x43434343u, hi ? 0x4342 : 0x4140);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x & 0x437F437Fu), "r"(x & 0x43804380u));
  } else {
    const uint32_t x = __byte_perm(w, 0u, hi ? 0x3424 : 0x1404);
    const uint32_t y = ((x & 0x7F007F00u) >> 4) | (x & 0x80008000u);
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(y), "r"(0x7B807B80u));  // 2^120
  }
  return r;
}

// mbar_wait for a kernel whose warps mostly wait: between tries the thread is
// suspended until the phase completes (or 20 us pass), and leaves the issue slots to the others.
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const uint32_t addr = smem_u32(bar);
  uint64_t since = 0;
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(addr), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    const uint64_t now = globaltimer_ns();
    if (since == 0) since = now;
    if (*abort || now - since > kWaitLimitNs) return false;
  }
}

template <int HD, int FMT, bool SPLITQ>
__global__ void __launch_bounds__(TcShape<HD, FMT, SPLITQ>::kThreads, 1) tree_attention_tc_kernel(const TreeArgs a) {
  using S = TcShape<HD, FMT, SPLITQ>;
  constexpr bool CODES = S::kCodes;
  constexpr int BK = S::kBK, RB = S::kRowBytes, CPR = RB / 16, NS = S::kStages, LG = S::kLoadGroups, NB = S::kBlocks, ROWS = S::kRows;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0u) {  // (there is no room to align it by hand)
    if (threadIdx.x == 0) atomicOr(a.err, kErrWaitTimeout);
    return;
  }
  TcBars& B = *reinterpret_cast<TcBars*>(smem + S::kBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&B.q_full, 4 * S::kQTiles + 2);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&B.k_full[i], kLoadWarps);
      mbar_init(&B.v_full[i], kLoadWarps);
      mbar_init(&B.k_empty[i], S::kQTiles);
      mbar_init(&B.v_empty[i], S::kQTiles);
    }
    for (int g = 0; g < 2; ++g)
      for (int i = 0; i < 2; ++i) {
        mbar_init(&B.s_full[g][i], 1);
        mbar_init(&B.p_full[g][i], 4);
        mbar_init(&B.pv_done[g][i], 1);
      }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&B.sums_full[i], 2);
      mbar_init(&B.taken[i], 2);
    }
    mbar_init(&B.drain[0], 1);
    mbar_init(&B.drain[1], 1);
    B.abort_flag = 0;
    B.odd_values = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    tmem_alloc(&B.tmem_base, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = B.tmem_base;  // S of group g: columns 128 g on; O of group g: 256 + HD g
  volatile int* abort_flag = &B.abort_flag;
  auto fail = [&] {
    *abort_flag = 1;
    atomicOr(a.err, kErrWaitTimeout);
  };
  // (every lane asks: one that asks for its warp and tells the others takes a tenth of the
  // kernel's time more)
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tc_wait(bar, parity, abort_flag)) != 0; };
  Walk<ROWS> w(a, blockIdx.x);
  uint32_t number = 0;  // of the segment's first tile: they are numbered over all segments

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax
    const int g = warp >> 2, qt = SPLITQ ? g : 0, row = (warp & 3) * 32 + lane;
    constexpr int STEP = SPLITQ ? 1 : 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t obase = tmem + lanes + 256 + g * HD;
    uint32_t j = 0, segment = 0, joined = 0;  // tiles, segments, and those whose sums were joined so far
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {  // (uniform over the warp)
      ok = warp_wait(bar, parity);
      return ok;
    };
    for (; ok && w.next(a); ++segment) {
      const int live = w.live_rows - qt * 128;  // rows of this query tile
      const int ntiles = (w.key1 - w.key0 + BK - 1) / BK;
      const uint32_t n0 = number;
      number += ntiles;
      const int row_all = w.row0 + qt * 128 + row;
      const bool exists = row < live;
      const int node = exists ? row_all / a.group : -1;
      const int head = w.kvh * a.group + (exists ? row_all - node * a.group : 0);
      const long long token = w.s.first + static_cast<long long>(exists ? node : 0);
      if (SPLITQ || g == 0) {
        if (exists) {
          const uint16_t* src = a.q + token * a.q_stride + head * HD;
          uint8_t* dst = smem + S::kQ + qt * NB * 16384 + row * 128;
#pragma unroll
          for (int c = 0; c < HD / 8; ++c)
            *reinterpret_cast<uint4*>(dst + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4)) = *reinterpret_cast<const uint4*>(src + 8 * c);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.q_full);
      }
      if (SPLITQ && live <= 0) {  // nothing in this query tile: its products are not issued
        // (not ahead of the others: a second arrival must not count for this segment)
        if (!wait(&B.q_full, segment & 1u)) break;
        continue;
      }
      const bool busy = (warp & 3) * 32 < live;  // (a warp without rows only keeps the barriers going)
      float m = kFirstMax, l = 0.f;
      bool any = false;  // O holds something
      for (int t = SPLITQ ? 0 : g; t < ntiles; t += STEP, ++j) {
        const int buf = j & 1;
        if (!wait(&B.s_full[g][buf], (j >> 1) & 1u)) break;
        if (busy) {
          tc_fence_after();
          const uint32_t sbase = tmem + lanes + 128 * g + (j & 1u) * BK;
          const float4* scales = reinterpret_cast<const float4*>(smem + S::kScale + ((n0 + t) % S::kScaleSlots) * 2 * BK * 4);
          const int base = w.key0 + t * BK;
          const bool partly = base + BK > min(w.ctx, w.key1);
          // P's buffer is free once the product that read it last is done. With two buffers that is
          // so already: the scores' product was issued behind it, and so is done after it.
          constexpr uint32_t PB = S::kPBufs;
          auto p_free = [&] { return PB == 2 || j < PB || wait(&B.pv_done[g][(j - PB) & 1], ((j - PB) >> 1) & 1u); };
          uint8_t* prow = smem + S::kP + (PB * g + j % PB) * S::kPBytes + row * 128;
          // Most tiles: every key is seen, and no score passes the maximum by more than
          // the slack. That is not waited for: the maximum stays as it is, and the tile is done
          // again, by the loop below, where a score turns out to pass it. Then nothing stands
          // between a score and its exponential, and the next 16 scores are under way meanwhile.
          auto quick = [&] {
            const unsigned long long up = f2_pack(a.scale_log2, a.scale_log2), minus_m = f2_pack(-m, -m);
            unsigned long long sum = f2_pack(0.f, 0.f), sum2 = sum;
            float worst = kFirstMax;
            uint32_t raw[2][16];
            tmem_ld_x16(sbase, raw[0]);
#pragma unroll
            for (int h = 0; h < BK / 16; ++h) {
              tmem_wait_ld();
              uint32_t(&now)[16] = raw[h & 1];
#pragma unroll
              for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(now[i]));  // (not used before the wait)
              if (h + 1 < BK / 16) tmem_ld_x16(sbase + 16 * (h + 1), raw[(h + 1) & 1]);
              float* sc = reinterpret_cast<float*>(now);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const unsigned long long f = CODES ? reinterpret_cast<const unsigned long long*>(scales)[8 * h + i] : up;
                f2_unpack(f2_fma(f2_pack(sc[2 * i], sc[2 * i + 1]), f, minus_m), sc[2 * i], sc[2 * i + 1]);
                worst = fmaxf(worst, fmaxf(sc[2 * i], sc[2 * i + 1]));
              }
              if (h == 0 && !p_free()) {
                tmem_wait_ld();
                return true;
              }
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                uint32_t e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int k = 8 * c + 2 * i;
                  unsigned long long p = f2_pack(ex2(sc[k]), ex2(sc[k + 1]));
                  if (i & 1)
                    sum2 = f2_add(sum2, p);
                  else
                    sum = f2_add(sum, p);
                  if constexpr (CODES) p = f2_mul(p, reinterpret_cast<const unsigned long long*>(scales)[BK / 2 + 8 * h + k / 2]);
                  float p0, p1;
                  f2_unpack(p, p0, p1);
                  e[i] = pack_rn_bf16x2(p0, p1);
                }
                *reinterpret_cast<uint4*>(prow + (h >> 2) * 16384 + (((2 * (h & 3) + c) ^ (row & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
              }
            }
            if (__any_sync(0xffffffffu, exists && worst > kSlack)) return false;
            float s0, s1;
            f2_unpack(f2_add(sum, sum2), s0, s1);
            l += s0 + s1;
            return true;
          };
          if (partly || !any || !quick()) {
            if (!p_free()) break;
            // Scores: raw where they take the scale with the exponent (bf16 cache,
            // positive scale), otherwise in units of log2; -inf where hidden.
            const bool late = !CODES && a.scale_log2 > 0.f;
            const float scale = late ? a.scale_log2 : 1.f;
            // 32 keys at a time, in a rolled loop: the roles' code together must not
            // outgrow the instruction cache.
#pragma unroll 1
            for (int h = 0; h < BK / 32; ++h) {
              uint32_t raw[32];
              float* sc = reinterpret_cast<float*>(raw);
              tmem_ld_x32(sbase + 32 * h, raw);
              tmem_wait_ld();
              if (!late) {
                const unsigned long long up = f2_pack(a.scale_log2, a.scale_log2);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const unsigned long long f = CODES ? reinterpret_cast<const unsigned long long*>(scales)[16 * h + i] : up;
                  f2_unpack(f2_mul(f2_pack(sc[2 * i], sc[2 * i + 1]), f), sc[2 * i], sc[2 * i + 1]);
                }
              }
              uint32_t seen = 0xFFFFFFFFu;
              if (partly) {
                const int k0 = base + 32 * h;
                seen = !exists ? 0u
                               : first_bits(w.key1 - k0) & (a.mask == nullptr
                                                                ? first_bits(w.ctx + node - k0 + 1)
                                                                : mask_window(a.mask + token * a.mask_words, a.mask_words, k0 - w.ctx));
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (!((seen >> i) & 1u)) sc[i] = -INFINITY;
              }
              float x4[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
              for (int i = 4; i < 28; i += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) x4[e] = fmaxf(x4[e], fmaxf(sc[i + e], sc[i + 4 + e]));
#pragma unroll
              for (int e = 0; e < 4; ++e) x4[e] = fmaxf(x4[e], sc[28 + e]);
              const float top = fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3])) * scale;
              // The maximum only takes whole values, so that what it moves is multiplied by powers of two.
              const bool move = exists && top > m + kSlack;
              if (__any_sync(0xffffffffu, move)) {
                const float to = move ? ceilf(top) : m;
                const float f = ex2(m - to);
                m = to;
                l *= f;
                if (any) {  // O holds the tiles before this one: wait for the last of them
                  if (!wait(&B.pv_done[g][buf ^ 1], ((j - 1) >> 1) & 1u)) break;
                  tc_fence_after();
#pragma unroll 1
                  for (int d = 0; d < HD; d += 16) {
                    uint32_t o[16];
                    tmem_ld_x16(obase + d, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tmem_st_x16(obase + d, o);
                  }
                  tmem_wait_st();
                }
                // and the probabilities in front of these
#pragma unroll 1
                for (int c = 0; c < 4 * h; ++c) {
                  uint4* q = reinterpret_cast<uint4*>(prow + (c >> 3) * 16384 + (((c & 7) ^ (row & 7)) << 4));
                  uint32_t e[4] = {q->x, q->y, q->z, q->w};
#pragma unroll
                  for (int i = 0; i < 4; ++i) e[i] = pack_rn_bf16x2(bf16lo(e[i]) * f, bf16hi(e[i]) * f);
                  *q = make_uint4(e[0], e[1], e[2], e[3]);
                }
              }
              unsigned long long sum = f2_pack(0.f, 0.f);
              const unsigned long long scale2 = f2_pack(scale, scale), minus_m = f2_pack(-m, -m);
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                uint32_t e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int k = 8 * c + 2 * i;
                  float p0, p1;
                  f2_unpack(f2_fma(f2_pack(sc[k], sc[k + 1]), scale2, minus_m), p0, p1);
                  p0 = ex2(p0);
                  p1 = ex2(p1);
                  sum = f2_add(sum, f2_pack(p0, p1));
                  if constexpr (CODES) {
                    f2_unpack(f2_mul(f2_pack(p0, p1), reinterpret_cast<const unsigned long long*>(scales)[BK / 2 + 16 * h + k / 2]), p0, p1);
                    if (partly) {  // (a hidden key's scale may be NaN)
                      if (!((seen >> k) & 1u)) p0 = 0.f;
                      if (!((seen >> (k + 1)) & 1u)) p1 = 0.f;
                    }
                  }
                  e[i] = pack_rn_bf16x2(p0, p1);
                }
                *reinterpret_cast<uint4*>(prow + (h >> 1) * 16384 + (((4 * (h & 1) + c) ^ (row & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
              }
              float s0, s1;
              f2_unpack(sum, s0, s1);
              l += s0 + s1;
            }
          }
          if (!ok) break;
        }
        any = true;
        tc_fence_before();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.p_full[g][buf]);
      }
      if (ok && any) wait(&B.pv_done[g][(j - 1) & 1], ((j - 1) >> 1) & 1u);
      if (!ok) break;
      if (!busy) continue;
      tc_fence_after();
      // ---- this row's sums: out, or its part of them. Where the groups had the same
      // rows, a row's values lie in the same lane of tensor memory: each group adds
      // up half of the columns.
      const bool whole = w.whole();
      constexpr int COLS = SPLITQ ? HD : HD / 2;
      const int d0 = SPLITQ ? 0 : g * COLS;
      float f0 = 1.f, f1 = 0.f;  // weights of this group's and the other one's values
      bool two = false;
      if constexpr (!SPLITQ) {
        float2* sums = reinterpret_cast<float2*>(smem + S::kSums) + row;
        sums[128 * g] = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.sums_full[warp & 3]);
        if (!wait(&B.sums_full[warp & 3], joined & 1u)) break;
        tc_fence_after();
        const float2 x = sums[0], y = sums[128];
        m = fmaxf(x.x, y.x);
        f0 = ex2(x.x - m);
        f1 = ex2(y.x - m);
        l = fmaf(x.y, f0, y.y * f1);
        two = ntiles > 1;  // (otherwise the second group had nothing)
      }
      // (behind the wait for the other group's sums: a group has waited for its own tiles only, and
      // writes columns of both groups' values)
      const bool odd = !CODES && *const_cast<volatile int*>(&B.odd_values) != 0;
      float* part = a.part + ((2ll * blockIdx.x + (w.u0 == 0 ? 1 : 0)) * ROWS + qt * 128 + row) * (HD + 4);
      uint16_t* out = a.out + token * a.out_stride + head * HD;
      const uint32_t o0 = SPLITQ ? obase : tmem + lanes + 256;
      // Rows are turned around in this warp's own piece of P, so that eight lanes store
      // 32 neighbouring columns of a row.
      const uint32_t turn = smem_u32(smem + S::kP) + g * S::kPBufs * S::kPBytes + (warp & 3) * 4096;
      const int rest = live - (warp & 3) * 32;  // rows of this warp
#pragma unroll 1
      for (int d = d0; d < d0 + COLS; d += 32) {
        uint32_t raw[32];
        float* o = reinterpret_cast<float*>(raw);
        tmem_ld_x32(o0 + d, raw);
        tmem_wait_ld();
        if (two) {
#pragma unroll
          for (int h = 0; h < 32; h += 16) {
            uint32_t more[16];
            tmem_ld_x16(o0 + HD + d + h, more);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[h + i] = o[h + i] * f0 + __uint_as_float(more[i]) * f1;
          }
        }
        if (odd && exists) {
          // (the keys of the tiles with new tokens)
          for (int k = w.key0 + (max(w.ctx - w.key0, 0) & ~(BK - 1)); k < w.key1; ++k) {
            const int n2 = k - w.ctx;
            if (!(a.mask == nullptr ? n2 <= node : (mask_window(a.mask + token * a.mask_words, a.mask_words, n2) & 1u) != 0u)) continue;
            const int page = __ldg(a.batch.page_table + w.b * a.batch.table_stride + (k >> a.pools.page_shift));
            if (page < 0 || page >= a.pools.num_pages) continue;
            const uint16_t* v = static_cast<const uint16_t*>(a.pools.v) +
                                kv_slot(a.pools, page, w.kvh, k & ((1 << a.pools.page_shift) - 1)) * HD + d;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if ((v[i] & 0x7F80u) == 0x7F80u) o[i] += bf16_to_f32(v[i]);
          }
        }
        const float f = whole ? out_factor(l, 0.f) : 1.f;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 8; ++c)
          sts128(turn + lane * 128 + ((c ^ (lane & 7)) << 4),
                 make_uint4(__float_as_uint(o[4 * c] * f), __float_as_uint(o[4 * c + 1] * f), __float_as_uint(o[4 * c + 2] * f),
                            __float_as_uint(o[4 * c + 3] * f)));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + (lane >> 3), c = lane & 7;
          const uint4 x = lds128(turn + r * 128 + ((c ^ (r & 7)) << 4));
          uint16_t* to = reinterpret_cast<uint16_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), r));
          if (r >= rest) continue;
          if (whole)
            *reinterpret_cast<uint2*>(to + d + 4 * c) = make_uint2(pack_rn_bf16x2(__uint_as_float(x.x), __uint_as_float(x.y)),
                                                                   pack_rn_bf16x2(__uint_as_float(x.z), __uint_as_float(x.w)));
          else
            *reinterpret_cast<uint4*>(part + (r - lane) * (HD + 4) + 4 + d + 4 * c) = x;
        }
      }
      if (exists && (SPLITQ || g == 0)) {
        if (!whole)
          *reinterpret_cast<float4*>(part) = make_float4(m, l, m, 0.f);
        else if (a.lse != nullptr)
          a.lse[token * a.heads + head] = lse_of(m, l);
      }
      tc_fence_before();
      __syncwarp();
      if constexpr (!SPLITQ) {
        // neither group's values nor its sums are overwritten before both have read them
        if (lane == 0) mbar_arrive(&B.taken[warp & 3]);
        if (!wait(&B.taken[warp & 3], joined & 1u)) break;
        ++joined;
      }
    }
    if (!ok) fail();
  } else if (warp < 10) {
    // ------------------------------------------- the products of one group each
    if (lane == 0) {
      const int g = warp - 8;
      constexpr uint32_t STEP = SPLITQ ? 1 : 2;
      const uint32_t id_s = tc_idesc(BK, false), id_o = tc_idesc(HD, true);
      const uint64_t dq = smem_desc_k_sw128(smem_u32(smem + S::kQ)) + (SPLITQ ? g * NB * 1024 : 0);
      const uint64_t dk = smem_desc_k_sw128(smem_u32(smem + S::kK));
      const uint64_t dp = smem_desc_k_sw128(smem_u32(smem + S::kP)) + g * (S::kPBufs * S::kPBytes / 16);
      const uint64_t dv = smem_desc_mn_sw128(smem_u32(smem + S::kV), S::kBlock);
      const uint32_t ts = tmem + 128 * g, to = tmem + 256 + g * HD;
      uint32_t js = 0, jo = 0, segment = 0;  // products issued, of each kind
      bool ok = true;
      auto s_ready = [&](uint32_t n) {
        // (P of the tile two before is there when its product was issued: so its scores were read)
        return js < jo + 2 && mbar_test_wait(&B.k_full[n % NS], (n / NS) & 1u);
      };
      auto issue_s = [&](uint32_t n) {
        const uint32_t st = n % NS, buf = js & 1u;
        tc_fence_after();
        const uint64_t db = dk + st * NB * (S::kBlock / 16);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          tc_mma_f16(ts + buf * BK, dq + (k >> 2) * 1024 + 2 * (k & 3), db + (k >> 2) * (S::kBlock / 16) + 2 * (k & 3), id_s, k != 0 ? 1u : 0u);
        tc_commit(&B.s_full[g][buf]);
        tc_commit(&B.k_empty[st]);
        ++js;
      };
      auto pv_ready = [&](uint32_t n) {
        return mbar_test_wait(&B.p_full[g][jo & 1], (jo >> 1) & 1u) && mbar_test_wait(&B.v_full[n % NS], (n / NS) & 1u);
      };
      auto issue_pv = [&](uint32_t n, bool first) {
        const uint32_t st = n % NS, buf = jo & 1u;
        tc_fence_after();
        const uint64_t da = dp + (jo % S::kPBufs) * (S::kPBytes / 16), db = dv + st * NB * (S::kBlock / 16);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) tc_mma_f16(to, da + 2 * k, db + k * 128, id_o, !first || k != 0 ? 1u : 0u);
        tc_commit(&B.pv_done[g][buf]);
        tc_commit(&B.v_empty[st]);
        ++jo;
      };
      for (; ok && w.next(a); ++segment) {
        const uint32_t ntiles = (w.key1 - w.key0 + BK - 1) / BK, n0 = number;
        number += ntiles;
        // (arrives as well as waits: a group without products in this segment would otherwise not be
        // waited for by anyone, and two segments late take one phase for another)
        mbar_arrive(&B.q_full);
        if (!(ok = tc_wait(&B.q_full, segment & 1u, abort_flag))) break;
        if (SPLITQ && w.live_rows <= 128 * g) {  // no rows: the tiles are only given back
          for (uint32_t n = n0; ok && n < number; ++n) {
            ok = tc_wait(&B.k_full[n % NS], (n / NS) & 1u, abort_flag) && tc_wait(&B.v_full[n % NS], (n / NS) & 1u, abort_flag);
            mbar_arrive(&B.k_empty[n % NS]);
            mbar_arrive(&B.v_empty[n % NS]);
          }
          continue;
        }
        // Whichever product can go next goes: the scores run ahead of the values' products
        // by up to two tiles, and neither waits for the other's operands.
        const uint32_t first = n0 + (SPLITQ ? 0 : g);
        uint32_t ns = first, no = first;
        uint64_t since = 0;
        uint32_t tries = 0;
        while (ok && no < number) {
          if (ns < number && s_ready(ns)) {
            issue_s(ns);
            ns += STEP;
          } else if (no < ns && pv_ready(no)) {
            issue_pv(no, no == first);
            no += STEP;
          } else {  // (bounded, as every wait here)
            if ((++tries & 63u) == 0u) {
              const uint64_t now = globaltimer_ns();
              if (since == 0) since = now;
              ok = !*abort_flag && now - since <= kWaitLimitNs;
            }
            continue;
          }
          since = 0;
        }
      }
      if (!ok) fail();
      // nothing of this group's is on its way to shared or tensor memory once this arrives
      tc_commit(&B.drain[g]);
      mbar_wait(&B.drain[g], 0, nullptr);
    }
  } else {
    // ------------------------------------------------------------------ loads
    const int group = (warp - 10) / kLoadWarps;
    const int tid = threadIdx.x - 32 * 10 - group * kLoadThreads;
    constexpr int PER = BK * CPR / kLoadThreads;  // 16-byte pieces of a thread, of K and of V: each KPX keys on
    constexpr int KPX = kLoadThreads / CPR;
    static_assert(KPX % 8 == 0, "a thread's pieces have one swizzle");
    const int page_mask = (1 << a.pools.page_shift) - 1;
    const int my_key = tid / CPR, my_c = tid % CPR;
    // A tile is asked for and handed over as one, or, where its places are few (128-wide bf16),
    // in parts: the keys' places are free long before the values'. us of one and two parts,
    // 128 rows of eight sequences: 86.7 and 81.4 at head_dim 128, 52.2 and 55.4 at 64.
    constexpr uint32_t PARTS = !CODES && HD == 128 ? 2 : 1, AHEAD = PARTS * S::kAhead;
    uint32_t issued = 0, done = 0;  // parts of this group's tiles: the numbers group, group + 2, ...
    uint32_t nodes = 0;             // bit i: the part issued i parts ago is of new tokens' values
    bool ok = true;
    // Pages of keys base + lane and base + 32 + lane of the next tile, asked for one tile
    // ahead of their use, and the places of those keys of this one (-1 behind the segment's
    // last key, or where the page is not there, which is reported).
    int page_lo = -1, page_hi = -1, lo = -1, hi = -1;
    auto ask_pages = [&](int base) {
      const int32_t* table = a.batch.page_table + w.b * a.batch.table_stride;
      page_lo = base + lane < w.key1 ? __ldg(table + ((base + lane) >> a.pools.page_shift)) : -1;
      page_hi = base + 32 + lane < w.key1 ? __ldg(table + ((base + 32 + lane) >> a.pools.page_shift)) : -1;
    };
    auto place_of = [&](int key, int page) {
      if (key >= w.key1) return -1;
      if (page < 0 || page >= a.pools.num_pages) {
        atomicOr(a.err, kErrBadIndex);
        return -1;
      }
      return static_cast<int>(kv_slot(a.pools, page, w.kvh, key & page_mask));
    };
    auto begin_tile = [&](int base, int next) {
      lo = place_of(base + lane, page_lo);
      hi = place_of(base + 32 + lane, page_hi);
      if (next < w.key1) ask_pages(next);
    };
    // asks for a part of tile n of the segment, the one at `base`
    auto issue = [&](uint32_t n, int base, uint32_t part) {
      const uint32_t at = CODES ? smem_u32(smem + S::kRawAt) + (n % (S::kRaw + !S::kRaw)) * 2 * BK * RB + tid * 16
                                : smem_u32(smem + S::kK) + ((n % NS) * NB + (my_c >> 3)) * S::kBlock + my_key * 128 + (((my_c & 7) ^ (my_key & 7)) << 4);
      constexpr uint32_t TO_X = CODES ? kLoadThreads * 16 : KPX * 128, TO_V = CODES ? BK * RB : S::kV - S::kK;
      const uint8_t* k = static_cast<const uint8_t*>(a.pools.k) + my_c * 16;
      const uint8_t* v = static_cast<const uint8_t*>(a.pools.v) + my_c * 16;
#pragma unroll
      for (int x = 0; x < PER; ++x) {  // (KPX divides 32: a piece's keys are all among the first 32, or all behind them)
        const int place = __shfl_sync(0xffffffffu, x * KPX < 32 ? lo : hi, (my_key + x * KPX) & 31);
        const long long byte = static_cast<long long>(max(place, 0)) * RB;
        if (PARTS == 1 || part == 0) cp16(at + x * TO_X, k + byte, place >= 0);
        if (PARTS == 1 || part == 1) cp16(at + TO_V + x * TO_X, v + byte, place >= 0);
      }
      if constexpr (CODES) {  // and scales: of key tid % 64, K's by the first 64 threads, V's by the others
        static_assert(2 * BK == kLoadThreads && BK == 64, "a scale a thread");
        const int place = (tid & 32) == 0 ? lo : hi;
        cp4(smem_u32(smem + S::kRawScale) + ((n % (S::kRaw + !S::kRaw)) * 2 * BK + tid) * 4,
            (tid < BK ? a.pools.k_scale : a.pools.v_scale) + max(place, 0), place >= 0);
      }
      cp_commit();
      nodes = nodes << 1 | (part == PARTS - 1 && base + BK > w.ctx ? 1u : 0u);
      ++issued;
    };
    // waits for the oldest part under way and hands it to the products
    auto finish = [&] {
      const uint32_t n = LG * (done / PARTS) + group;
      const int st = n % NS;
      if (issued - done == AHEAD)
        cp_wait<AHEAD - 1>();
      else
        cp_wait<0>();
      if constexpr (CODES) {
        const float scale = reinterpret_cast<const float*>(smem + S::kRawScale)[(n % (S::kRaw + !S::kRaw)) * 2 * BK + tid];
        reinterpret_cast<float*>(smem + S::kScale)[(n % S::kScaleSlots) * 2 * BK + tid] = tid < BK ? scale * a.scale_log2 : scale;
        const uint32_t from = smem_u32(smem + S::kRawAt) + (n % (S::kRaw + !S::kRaw)) * 2 * BK * RB + tid * 16;
        const uint32_t to = smem_u32(smem + S::kK) + (st * NB + (my_c >> 2)) * S::kBlock + my_key * 128;
        // (128-wide rows: half of the lanes store their second eight values first, so that a
        // row's pieces in both 64-dim columns lie in different banks)
        const uint32_t flip = HD == 128 ? my_c >> 2 & 1 : 0;
        const uint32_t to0 = (((2 * my_c + flip) & 7) ^ (my_key & 7)) << 4, to1 = to0 ^ 16u;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          if (n >= NS && !warp_wait(kv ? &B.v_empty[st] : &B.k_empty[st], ((n / NS) - 1) & 1u)) return false;
          uint4 raw[PER];
#pragma unroll
          for (int x = 0; x < PER; ++x) raw[x] = lds128(from + kv * BK * RB + x * kLoadThreads * 16);
#pragma unroll
          for (int x = 0; x < PER; ++x) {
            const uint4 v = raw[x];
            const uint32_t e[4] = {flip ? v.z : v.x, flip ? v.w : v.y, flip ? v.x : v.z, flip ? v.y : v.w};
            uint32_t o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[2 * i] = code_pair_bf16<FMT>(e[i], 0);
              o[2 * i + 1] = code_pair_bf16<FMT>(e[i], 1);
            }
            const uint32_t dst = to + (kv ? S::kV - S::kK : 0) + x * KPX * 128;
            sts128(dst + to0, make_uint4(o[0], o[1], o[2], o[3]));
            sts128(dst + to1, make_uint4(o[4], o[5], o[6], o[7]));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(kv ? &B.v_full[st] : &B.k_full[st]);
        }
      } else {
        if ((nodes >> (issued - done - 1)) & 1u) {
          const uint32_t at = smem_u32(smem + S::kV) + (st * NB + (my_c >> 3)) * S::kBlock + my_key * 128 + (((my_c & 7) ^ (my_key & 7)) << 4);
#pragma unroll 1
          for (int x = 0; x < PER; ++x) {
            const uint4 v = lds128(at + x * KPX * 128);
            uint32_t e[4] = {v.x, v.y, v.z, v.w};
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((e[i] & 0x7F80u) == 0x7F80u) e[i] &= 0xFFFF0000u, odd = true;
              if ((e[i] & 0x7F800000u) == 0x7F800000u) e[i] &= 0x0000FFFFu, odd = true;
            }
            if (odd) {
              sts128(at + x * KPX * 128, make_uint4(e[0], e[1], e[2], e[3]));
              atomicExch(&B.odd_values, 1);
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (PARTS == 1 || done % PARTS == 0) mbar_arrive(&B.k_full[st]);
          if (PARTS == 1 || done % PARTS == 1) mbar_arrive(&B.v_full[st]);
        }
      }
      ++done;
      return true;
    };
    while (ok && w.next(a)) {
      const int ntiles = (w.key1 - w.key0 + BK - 1) / BK;
      const uint32_t first = number;
      number += ntiles;
      const int t0 = (group - first) & (LG - 1);
      ask_pages(w.key0 + t0 * BK);
      for (int t = t0; ok && t < ntiles; t += LG) {
        const uint32_t n = first + t;
        begin_tile(w.key0 + t * BK, w.key0 + (t + LG) * BK);
#pragma unroll 1
        for (uint32_t part = 0; ok && part < PARTS; ++part) {
          if (issued - done == AHEAD) ok = finish();
          if constexpr (!CODES) {
            // The place's last tile must be done with. Where it is not yet, the parts under way
            // are handed over first: the products may be waiting for just those.
            if (ok && n >= NS) {
              // (a tile's values are done with after its keys)
              uint64_t* bar = PARTS == 2 && part == 0 ? &B.k_empty[n % NS] : &B.v_empty[n % NS];
              const uint32_t parity = ((n / NS) - 1) & 1u;
              auto free_now = [&] { return __all_sync(0xffffffffu, mbar_test_wait(bar, parity)) != 0; };
              while (ok && done < issued && !free_now()) ok = finish();
              ok = ok && warp_wait(bar, parity);
              if (PARTS == 1) ok = ok && warp_wait(&B.k_empty[n % NS], parity);
            }
          }
          if (ok) issue(n, w.key0 + t * BK, part);
        }
      }
    }
    while (ok && done < issued) ok = finish();
    cp_wait<0>();
    if (!ok) fail();
  }
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, S::kTmemCols);
}

template <int HD, int FMT, bool SPLITQ>
TreeTcVariant tc_variant() {
  using S = TcShape<HD, FMT, SPLITQ>;
  return TreeTcVariant{tree_attention_tc_kernel<HD, FMT, SPLITQ>, S::kRows, S::kThreads, S::kSmem};
}

template <int FMT>
TreeTcVariant tc_variant_of(int head_dim, int64_t rows) {
  if (head_dim == 128) return tc_variant<128, FMT, false>();
  return rows <= 128 ? tc_variant<64, FMT, false>() : tc_variant<64, FMT, true>();
}

}  // namespace

TreeTcVariant tree_tc_variant(int format, int head_dim, int64_t rows) {
  return format == NCM_KV_BF16   ? tc_variant_of<NCM_KV_BF16>(head_dim, rows)
         : format == NCM_KV_INT8 ? tc_variant_of<NCM_KV_INT8>(head_dim, rows)
                                 : tc_variant_of<NCM_KV_E4M3>(head_dim, rows);
}

}  // namespace ncm
