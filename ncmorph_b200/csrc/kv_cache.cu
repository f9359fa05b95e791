// The paged key/value cache: ncm_kv_cache_append (quantised as it is written)
// and ncm_kv_cache_gather (read back as bf16 rows).
//
// A head's row of one token (head_dim bf16 values) belongs to head_dim / 8
// neighbouring lanes, eight values each. Written, per row with A = max |x|:
//   code = round(M x / A), scale = A / M, M = 127 (int8) or 448 (e4m3).
// A quotient M x / A that is not halfway between two codes is off from halfway
// by 2^-16 or more, relative to itself: M x and A have at most 15 and 8
// significant bits, so their nonzero differences from a halfway point are
// whole units of at most 16 bits (13 for e4m3, whose halfway points have 5 bits).
// x * (M * rcp(A)) is off by 2^-21 at most. Rounded to 18 bits (Veltkamp's splitting) it is
// halfway exactly where the quotient is, so the codes are those of exact
// arithmetic, ties included, without a division per value.
//
// Bound: memory; no value is used twice. 16 thousand tokens of 8 heads of 128: written
// as bf16 in 26.3 us (5.1 TB/s moved), as int8 or e4m3 in 26.7 (3.8 TB/s): the same time
// for fewer bytes. Rows are asked for once their slots are known, and 44 (60) registers leave
// five (four) blocks an SM, so too few bytes are on their way; ALU and issue slots are half
// idle. Read back in 19-22 us. Contexts of 16 sequences of up to 16384 tokens, 8 heads of 64,
// int8: read back in 53 us, 5.4 TB/s, 0.83 of a copy.
#include <algorithm>

#include "kv_cache.cuh"

namespace ncm {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowTokens = 16;  // rows of a chunk at most

__device__ __forceinline__ uint16_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

__device__ __forceinline__ float2 f16x2_to_f32(uint32_t v) {
  float2 r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "r"(v));
  return r;
}

// The largest magnitude of a row held by LPR lanes, as bf16 bits (they order as integers).
template <int LPR>
__device__ __forceinline__ uint32_t row_top(const uint4& v) {
  uint32_t top = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
  return max(top >> 16, top & 0xFFFFu);
}

// Eight values of a row whose largest magnitude is `top` -> their codes and the row's scale.
template <int FMT>
__device__ __forceinline__ uint2 quantise8(const uint4& v, uint32_t top, float* scale) {
  constexpr float M = FMT == NCM_KV_INT8 ? 127.f : 448.f;
  const uint32_t e[4] = {v.x, v.y, v.z, v.w};
  const float big = __uint_as_float(top << 16);
  float y[8], factor;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = (i & 1) ? bf16hi(e[i >> 1]) : bf16lo(e[i >> 1]);
  if (top - 0x1000u < 0x6E80u) {  // 2^-95 <= A < 2^126: 1 / A and M / A are normal numbers
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(big));
    factor = M * inv;
    // A / M: one correction by the exact remainder rounds it correctly (A has 128 mantissas)
    const float q = big * (1.f / M);
    *scale = fmaf(fmaf(-q, M, big), 1.f / M, q);
  } else if (top == 0u || top >= 0x7F80u) {  // zeros; a NaN or an infinity
    *scale = top == 0u ? 1.f : __uint_as_float(0x7FC00000u);
    return make_uint2(0u, 0u);
  } else {
    const float pre = top < 0x1000u ? 0x1p64f : 0x1p-32f;
    *scale = __fdiv_rn(big, M);
    factor = __fdiv_rn(M, big * pre);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= pre;
  }
  const unsigned long long f2 = f2_pack(factor, factor), s2 = f2_pack(65.f, 65.f), n2 = f2_pack(-1.f, -1.f);
#pragma unroll
  for (int i = 0; i < 8; i += 2) {  // q = y factor rounded to 18 bits: c - (c - q) with c = 65 q
    const unsigned long long q = f2_mul(f2_pack(y[i], y[i + 1]), f2), c = f2_mul(q, s2);
    unsigned long long r = f2_fma(f2_fma(q, n2, c), n2, c);
    // 1.5 * 2^23 + q rounds q to a whole number, ties to even; its low byte is the code
    if constexpr (FMT == NCM_KV_INT8) r = f2_add(r, f2_pack(12582912.f, 12582912.f));
    f2_unpack(r, y[i], y[i + 1]);
  }
  uint32_t out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (FMT == NCM_KV_INT8) {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(y[4 * h + i]);
      out[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
      out[h] = pack_e4m3x2(y[4 * h], y[4 * h + 1]) | (static_cast<uint32_t>(pack_e4m3x2(y[4 * h + 2], y[4 * h + 3])) << 16);
    }
  }
  return make_uint2(out[0], out[1]);
}

template <int FMT>
__device__ __forceinline__ uint4 dequantise8(uint32_t lo, uint32_t hi, float scale) {
  const uint32_t w[2] = {lo, hi};
  const unsigned long long s2 = f2_pack(scale, scale);
  uint32_t out[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    unsigned long long y;
    if constexpr (FMT == NCM_KV_INT8) {  // 2^23 + 128 + code, less 2^23 + 128
      const uint32_t x = w[h >> 1] ^ 0x80808080u;
      y = f2_add(f2_pack(__uint_as_float(__byte_perm(x, 0x4B000000u, 0x7440 | (2 * (h & 1)))),
                         __uint_as_float(__byte_perm(x, 0x4B000000u, 0x7440 | (2 * (h & 1) + 1)))),
                 f2_pack(-8388736.f, -8388736.f));
    } else {
      const float2 a = f16x2_to_f32(e4m3x2_to_f16x2(static_cast<uint16_t>(w[h >> 1] >> (16 * (h & 1)))));
      y = f2_pack(a.x, a.y);
    }
    float p, q;
    f2_unpack(f2_mul(y, s2), p, q);
    out[h] = pack_rn_bf16x2(p, q);
  }
  return make_uint4(out[0], out[1], out[2], out[3]);
}

struct RowsArgs {
  KvPools pools;
  KvBatch batch;
  const int32_t* begin;  // gather: first position of each sequence, or null
  uint16_t* k;           // the caller's rows (append only reads them)
  uint16_t* v;
  long long k_stride, v_stride;
  int tokens;     // rows of one block, at most kRowTokens
  int part_rows;  // head rows that a block's threads hold at a time
  int* err;
};

// Slot of packed row t (page * page_size + offset), or -1 where there is none:
// behind the last sequence, or in a sequence or page that does not fit, which is reported.
template <bool APPEND>
__device__ __forceinline__ int slot_of_row(const RowsArgs& a, long long t) {
  if (t >= a.batch.rows) return -1;
  const int b = sequence_of_row(a.batch.token_start, a.batch.batch, t);
  if (b < 0) return -1;
  const int first = __ldg(a.batch.token_start + b), n = __ldg(a.batch.token_start + b + 1) - first;
  int begin;
  if (APPEND) {
    const int len = __ldg(a.batch.kv_lens + b);
    begin = len < n ? -1 : len - n;
  } else {
    begin = a.begin != nullptr ? __ldg(a.begin + b) : 0;
  }
  // a sequence that does not fit is skipped as a whole
  if (first < 0 || begin < 0 || static_cast<long long>(begin) + n > kv_capacity(a.batch, a.pools) ||
      static_cast<long long>(first) + n > a.batch.rows) {
    atomicOr(a.err, kErrBadIndex);
    return -1;
  }
  const int pos = begin + static_cast<int>(t - first);
  const int page = __ldg(a.batch.page_table + b * a.batch.table_stride + (pos >> a.pools.page_shift));
  if (page < 0 || page >= a.pools.num_pages) {
    atomicOr(a.err, kErrBadIndex);
    return -1;
  }
  return (page << a.pools.page_shift) + (pos & ((1 << a.pools.page_shift) - 1));
}

// Reports sequences that no row of the call leads to, but whose rows are not there: past the
// end, or fewer than none. By threads that have no slot to look up, while others do.
__device__ __forceinline__ void check_sequences(const RowsArgs& a) {
  constexpr unsigned kCheckers = kRowThreads - 32;
  if (blockIdx.y != 0 || threadIdx.x < 32) return;
  const int rows = static_cast<int>(a.batch.rows);
#pragma unroll 1
  for (unsigned b = blockIdx.x * kCheckers + threadIdx.x - 32; b < static_cast<unsigned>(a.batch.batch); b += gridDim.x * kCheckers) {
    const int first = __ldg(a.batch.token_start + b), end = __ldg(a.batch.token_start + b + 1);
    if (end < first || (end > first && (first < 0 || end > rows))) atomicOr(a.err, kErrBadIndex);
  }
}

// A block moves chunks of `tokens` rows: one lane each resolves the next chunk's
// slots while this one's rows are on their way. A thread keeps its eight values
// of a row (a head of the keys or the values: blockIdx.y picks the part of the
// row) and walks over the chunk's rows, BATCH of them loaded before the first is stored.
template <int FMT, int HD, bool APPEND>
__global__ void __launch_bounds__(kRowThreads) kv_rows_kernel(const RowsArgs a) {
  __shared__ int slot_of[2][kRowTokens];
  pdl_wait();
  pdl_launch_dependents();
  constexpr bool CODES = FMT != NCM_KV_BF16;
  constexpr int LPR = HD / 8, EB = CODES ? 1 : 2, BATCH = APPEND ? 4 : 2;
  const int lane_row = threadIdx.x / LPR, piece = threadIdx.x % LPR;
  const int e = blockIdx.y * a.part_rows + lane_row % a.part_rows;  // head row: keys, then values
  const int first = lane_row / a.part_rows, step = (kRowThreads / LPR) / a.part_rows;  // this thread's tokens
  const bool idle = e >= 2 * a.pools.kv_heads || first >= step;
  const bool is_v = e >= a.pools.kv_heads;
  const int h = is_v ? e - a.pools.kv_heads : e;
  const long long stride = is_v ? a.v_stride : a.k_stride;
  uint8_t* codes = static_cast<uint8_t*>(is_v ? a.pools.v : a.pools.k) + piece * 8 * EB;
  float* scales = is_v ? a.pools.v_scale : a.pools.k_scale;
  long long t0 = static_cast<long long>(blockIdx.x) * a.tokens;
  const long long t_step = static_cast<long long>(gridDim.x) * a.tokens;
  if (threadIdx.x < a.tokens) slot_of[0][threadIdx.x] = slot_of_row<APPEND>(a, t0 + threadIdx.x);
  check_sequences(a);
  __syncthreads();
  for (int turn = 0; t0 < a.batch.rows; t0 += t_step, turn ^= 1) {
    const int* slots = slot_of[turn];
    uint16_t* rows = (is_v ? a.v : a.k) + t0 * stride + h * HD + piece * 8;
    if (threadIdx.x < a.tokens) slot_of[turn ^ 1][threadIdx.x] = slot_of_row<APPEND>(a, t0 + t_step + threadIdx.x);
    for (int i0 = 0; i0 < a.tokens; i0 += BATCH * step) {
      uint4 x[BATCH];
      float scale[BATCH];
      long long at[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int i = i0 + k * step + first;
        const int slot = !idle && i < a.tokens ? slots[i] : -1;
        at[k] = slot < 0 ? -1 : kv_slot(a.pools, slot >> a.pools.page_shift, h, slot & ((1 << a.pools.page_shift) - 1));
        x[k] = make_uint4(0u, 0u, 0u, 0u);
        if (at[k] < 0) continue;
        if constexpr (APPEND) {
          x[k] = __ldcs(reinterpret_cast<const uint4*>(rows + i * stride));
        } else if constexpr (CODES) {
          const uint2 c = *reinterpret_cast<const uint2*>(codes + at[k] * HD);
          x[k].x = c.x;
          x[k].y = c.y;
          scale[k] = scales[at[k]];
        } else {
          x[k] = *reinterpret_cast<const uint4*>(codes + at[k] * (HD * EB));
        }
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        uint16_t* row = rows + (i0 + k * step + first) * stride;
        if constexpr (APPEND && CODES) {
          const uint32_t top = row_top<LPR>(x[k]);
          if (at[k] >= 0) {
            float sc;
            *reinterpret_cast<uint2*>(codes + at[k] * HD) = quantise8<FMT>(x[k], top, &sc);
            if (piece == 0) scales[at[k]] = sc;
          }
        } else if (at[k] >= 0) {
          if constexpr (APPEND)
            *reinterpret_cast<uint4*>(codes + at[k] * (HD * EB)) = x[k];
          else if constexpr (CODES)
            *reinterpret_cast<uint4*>(row) = dequantise8<FMT>(x[k].x, x[k].y, scale[k]);
          else
            *reinterpret_cast<uint4*>(row) = x[k];
        }
      }
    }
    __syncthreads();
  }
}

template <bool APPEND>
int launch_rows(ncm_ctx* ctx, const ncm_kv_cache_t* c, RowsArgs& a, cudaStream_t st) {
  // Few rows: a block each, so that they reach every SM. Many: up to kRowTokens a
  // block, which looks their slots up together.
  a.tokens = static_cast<int>(std::min<int64_t>(kRowTokens, std::max<int64_t>(1, a.batch.rows / (4 * ctx->num_sms))));
  a.part_rows = std::min(2 * c->kv_heads, kRowThreads / (c->head_dim / 8));
  const int parts = ceil_div(2 * c->kv_heads, a.part_rows);
  const int blocks = std::min(ceil_div(a.batch.rows, a.tokens), std::max(1, 8 * ctx->num_sms / parts));
  a.err = ctx->d_err;
  using Kernel = void (*)(const RowsArgs);
  static const Kernel table[3][2] = {
      {kv_rows_kernel<NCM_KV_BF16, 64, APPEND>, kv_rows_kernel<NCM_KV_BF16, 128, APPEND>},
      {kv_rows_kernel<NCM_KV_INT8, 64, APPEND>, kv_rows_kernel<NCM_KV_INT8, 128, APPEND>},
      {kv_rows_kernel<NCM_KV_E4M3, 64, APPEND>, kv_rows_kernel<NCM_KV_E4M3, 128, APPEND>}};
  Launch _launch(ctx, KID_KV_CACHE, st);
  NCM_CUDA_TRY(launch_pdl(table[c->format][c->head_dim == 128], dim3(blocks, parts), dim3(kRowThreads), 0, st, 1, a));
  return NCM_OK;
}

// Whether row arrays a and b of equal width share an element (strides in elements). Column
// slices of the same rows do not; other strides than each other's over one range are taken to.
bool rows_overlap(const uint16_t* a, int64_t a_stride, const uint16_t* b, int64_t b_stride, int64_t rows, int64_t width) {
  if (!ranges_overlap(a, 2 * ((rows - 1) * a_stride + width), b, 2 * ((rows - 1) * b_stride + width))) return false;
  if (a_stride != b_stride) return true;
  const int64_t at = (a < b ? b - a : a - b) % a_stride;
  return at < width || at + width > a_stride;
}

int rows_args(const char* what, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, bool need_lens,
              const uint16_t* k, int64_t k_stride, const uint16_t* v, int64_t v_stride, RowsArgs* a) {
  int rc = kv_check_cache(what, cache);
  if (rc || (rc = kv_check_batch(what, batch, need_lens))) return rc;
  const int64_t width = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
  if ((rc = kv_check_rows(what, "k", k, k_stride, batch->rows, width)) ||
      (rc = kv_check_rows(what, "v", v, v_stride, batch->rows, width)))
    return rc;
  const size_t pool = static_cast<size_t>(cache->num_pages) * cache->page_size * width * (cache->format == NCM_KV_BF16 ? 2 : 1);
  for (const void* p : {cache->k, cache->v})
    if (batch->rows > 0 && (ranges_overlap(k, 2 * ((batch->rows - 1) * k_stride + width), p, pool) ||
                            ranges_overlap(v, 2 * ((batch->rows - 1) * v_stride + width), p, pool)))
      return ncm_fail(NCM_EINVAL, "%s: the rows overlap a pool", what);
  a->pools = kv_pools_of(cache);
  a->batch = kv_batch_of(batch);
  a->k = const_cast<uint16_t*>(k);
  a->v = const_cast<uint16_t*>(v);
  a->k_stride = k_stride;
  a->v_stride = v_stride;
  return NCM_OK;
}

}  // namespace
}  // namespace ncm

using namespace ncm;

extern "C" {

int ncm_kv_cache_append(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, const uint16_t* k,
                        int64_t k_stride, const uint16_t* v, int64_t v_stride, ncm_stream_t stream) {
  DeviceGuard guard(ctx);
  if (guard.status()) return guard.status();
  RowsArgs a{};
  int rc = rows_args("kv_cache_append", cache, batch, true, k, k_stride, v, v_stride, &a);
  if (rc || batch->batch == 0 || batch->rows == 0) return rc;
  return launch_rows<true>(ctx, cache, a, static_cast<cudaStream_t>(stream));
}

int ncm_kv_cache_gather(ncm_ctx_t* ctx, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, const int32_t* begin,
                        uint16_t* k, int64_t k_stride, uint16_t* v, int64_t v_stride, ncm_stream_t stream) {
  DeviceGuard guard(ctx);
  if (guard.status()) return guard.status();
  RowsArgs a{};
  int rc = rows_args("kv_cache_gather", cache, batch, false, k, k_stride, v, v_stride, &a);
  if (rc || batch->batch == 0 || batch->rows == 0) return rc;
  if (!aligned_to(begin, 4)) return ncm_fail(NCM_EINVAL, "kv_cache_gather: misaligned begin");
  if (rows_overlap(k, k_stride, v, v_stride, batch->rows, static_cast<int64_t>(cache->kv_heads) * cache->head_dim))
    return ncm_fail(NCM_EINVAL, "kv_cache_gather: the rows of k and v overlap");
  a.begin = begin;
  return launch_rows<false>(ctx, cache, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
