// The paged key/value cache: ncm_kv_cache_append (quantised as it is written)
// and ncm_kv_cache_gather (read back as bf16 rows).
//
// A head's row of one token (head_dim bf16 values) belongs to head_dim / 8
// neighbouring lanes, eight values each. Written, per row with A = max |x|:
//   code = round(M x / A), scale = A / M, M = 127 (int8) or 448 (e4m3).
// M x is exact in f32 (bf16 has 8 significant bits, M at most 7) and the
// quotient is correctly rounded. A quotient that is not halfway between two
// codes is off from halfway by at least 2^-17 of a code at the top of the
// range (its numerator and A are integers of at most 15 and 8 bits), which is
// more than its rounding error of 2^-18, so the codes are those of exact arithmetic.
//
// Bound: memory; no value is used twice.
#include <algorithm>

#include "kv_cache.cuh"

namespace ncm {
namespace {

constexpr int kRowThreads = 256;

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

// Eight values of a row -> its eight codes and the row's scale. LPR lanes hold the row.
template <int FMT, int LPR>
__device__ __forceinline__ uint2 quantise8(const uint4& v, float* scale) {
  const uint32_t e[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;  // the largest magnitude, as bf16 bits (they order as integers)
#pragma unroll
  for (int i = 0; i < 4; ++i) top = max(top, max(e[i] & 0x7FFFu, (e[i] >> 16) & 0x7FFFu));
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  constexpr float M = FMT == NCM_KV_INT8 ? 127.f : 448.f;
  if (top >= 0x7F80u) {
    *scale = __uint_as_float(0x7FC00000u);
    return make_uint2(0u, 0u);
  }
  if (top == 0) {
    *scale = 1.f;
    return make_uint2(0u, 0u);
  }
  float big = __uint_as_float(top << 16);
  *scale = __fdiv_rn(big, M);
  // M x must not overflow: rows this large are brought down by a power of two first
  const float f = top >= 0x7000u ? 0x1p-32f : 1.f;
  big *= f;
  float y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = __fdiv_rn(bf16lo(e[i]) * f * M, big);
    y[2 * i + 1] = __fdiv_rn(bf16hi(e[i]) * f * M, big);
  }
  uint32_t out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (FMT == NCM_KV_INT8) {
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= (static_cast<uint32_t>(__float2int_rn(y[4 * h + i])) & 0xFFu) << (8 * i);
      out[h] = w;
    } else {
      out[h] = pack_e4m3x2(y[4 * h], y[4 * h + 1]) | (static_cast<uint32_t>(pack_e4m3x2(y[4 * h + 2], y[4 * h + 3])) << 16);
    }
  }
  return make_uint2(out[0], out[1]);
}

template <int FMT>
__device__ __forceinline__ uint4 dequantise8(const uint2& c, float scale) {
  float y[8];
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (FMT == NCM_KV_INT8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[4 * h + i] = static_cast<float>(static_cast<int8_t>(w[h] >> (8 * i)));
    } else {
      const float2 a = f16x2_to_f32(e4m3x2_to_f16x2(static_cast<uint16_t>(w[h])));
      const float2 b = f16x2_to_f32(e4m3x2_to_f16x2(static_cast<uint16_t>(w[h] >> 16)));
      y[4 * h] = a.x;
      y[4 * h + 1] = a.y;
      y[4 * h + 2] = b.x;
      y[4 * h + 3] = b.y;
    }
  }
  return make_uint4(pack_bf16x2(y[0] * scale, y[1] * scale), pack_bf16x2(y[2] * scale, y[3] * scale),
                    pack_bf16x2(y[4] * scale, y[5] * scale), pack_bf16x2(y[6] * scale, y[7] * scale));
}

struct RowsArgs {
  KvPools pools;
  KvBatch batch;
  const int32_t* begin;  // gather: first position of each sequence, or null
  uint16_t* k;           // the caller's rows (append only reads them)
  uint16_t* v;
  long long k_stride, v_stride;
  int parts;        // warp-wide steps of one token's rows (its key heads, then its value heads)
  int token_warps;  // warps that share one token
  int* err;
};

// One warp per (token, share of its parts). In a step the warp's 32 lanes move
// 32 / LPR head rows.
template <int FMT, int HD, bool APPEND>
__global__ void __launch_bounds__(kRowThreads) kv_rows_kernel(const RowsArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int LPR = HD / 8, RPS = 32 / LPR, EB = FMT == NCM_KV_BF16 ? 2 : 1;
  const int lane = threadIdx.x & 31;
  const long long warp = static_cast<long long>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5);
  const long long t = warp / a.token_warps;
  const int share = static_cast<int>(warp - t * a.token_warps);
  if (t >= a.batch.rows) return;
  const int b = sequence_of_row(a.batch.token_start, a.batch.batch, t);
  if (b < 0) return;
  const int first = __ldg(a.batch.token_start + b), n = __ldg(a.batch.token_start + b + 1) - first;
  int begin;
  if (APPEND) {
    const int len = __ldg(a.batch.kv_lens + b);
    begin = len < n ? -1 : len - n;
  } else {
    begin = a.begin != nullptr ? __ldg(a.begin + b) : 0;
  }
  const long long cap = static_cast<long long>(a.batch.table_width) << a.pools.page_shift;
  // a sequence that does not fit is skipped as a whole
  if (first < 0 || begin < 0 || static_cast<long long>(begin) + n > cap ||
      static_cast<long long>(first) + n > a.batch.rows) {
    if (lane == 0) atomicOr(a.err, kErrBadIndex);
    return;
  }
  const int pos = begin + static_cast<int>(t - first);
  const int page = __ldg(a.batch.page_table + b * a.batch.table_stride + (pos >> a.pools.page_shift));
  if (page < 0 || page >= a.pools.num_pages) {
    if (lane == 0) atomicOr(a.err, kErrBadIndex);
    return;
  }
  const int off = pos & ((1 << a.pools.page_shift) - 1);
  const int piece = lane % LPR;
#pragma unroll 4
  for (int p = share; p < a.parts; p += a.token_warps) {
    const int r = p * RPS + lane / LPR;
    const bool live = r < 2 * a.pools.kv_heads;
    const bool is_v = r >= a.pools.kv_heads;
    const int h = is_v ? r - a.pools.kv_heads : r;
    uint16_t* row = (is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride) + h * HD + piece * 8;
    const long long slot = kv_slot(a.pools, page, h, off);
    uint8_t* code = static_cast<uint8_t*>(is_v ? a.pools.v : a.pools.k) + (slot * HD + piece * 8) * EB;
    float* scales = is_v ? a.pools.v_scale : a.pools.k_scale;
    if constexpr (APPEND) {
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if (live) x = *reinterpret_cast<const uint4*>(row);
      if constexpr (FMT == NCM_KV_BF16) {
        if (live) *reinterpret_cast<uint4*>(code) = x;
      } else {
        float scale;
        const uint2 c = quantise8<FMT, LPR>(x, &scale);
        if (live) {
          *reinterpret_cast<uint2*>(code) = c;
          if (piece == 0) scales[slot] = scale;
        }
      }
    } else if (live) {
      if constexpr (FMT == NCM_KV_BF16)
        *reinterpret_cast<uint4*>(row) = *reinterpret_cast<const uint4*>(code);
      else
        *reinterpret_cast<uint4*>(row) = dequantise8<FMT>(*reinterpret_cast<const uint2*>(code), scales[slot]);
    }
  }
}

template <bool APPEND>
int launch_rows(ncm_ctx* ctx, const ncm_kv_cache_t* c, RowsArgs& a, cudaStream_t st) {
  const int lpr = c->head_dim / 8;
  a.parts = ceil_div(2 * c->kv_heads, 32 / lpr);
  // Few tokens: a warp for each part, so that the call is one step long. Many:
  // one warp a token, which looks its sequence and page up once.
  a.token_warps = a.batch.rows * a.parts <= 8 * static_cast<long long>(ctx->num_sms) ? a.parts : 1;
  a.err = ctx->d_err;
  using Kernel = void (*)(const RowsArgs);
  static const Kernel table[3][2] = {
      {kv_rows_kernel<NCM_KV_BF16, 64, APPEND>, kv_rows_kernel<NCM_KV_BF16, 128, APPEND>},
      {kv_rows_kernel<NCM_KV_INT8, 64, APPEND>, kv_rows_kernel<NCM_KV_INT8, 128, APPEND>},
      {kv_rows_kernel<NCM_KV_E4M3, 64, APPEND>, kv_rows_kernel<NCM_KV_E4M3, 128, APPEND>}};
  Launch _launch(ctx, KID_KV_CACHE, st);
  NCM_CUDA_TRY(launch_pdl(table[c->format][c->head_dim == 128], dim3(ceil_div(a.batch.rows * a.token_warps, kRowThreads / 32)),
                          dim3(kRowThreads), 0, st, 1, a));
  return NCM_OK;
}

int rows_args(const char* what, const ncm_kv_cache_t* cache, const ncm_kv_batch_t* batch, bool need_lens,
              const uint16_t* k, int64_t k_stride, const uint16_t* v, int64_t v_stride, RowsArgs* a) {
  int rc = kv_check_cache(what, cache);
  if (rc || (rc = kv_check_batch(what, batch, need_lens))) return rc;
  const int64_t width = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
  if ((rc = kv_check_rows(what, "k", k, k_stride, batch->rows, width)) ||
      (rc = kv_check_rows(what, "v", v, v_stride, batch->rows, width)))
    return rc;
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
  a.begin = begin;
  return launch_rows<false>(ctx, cache, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
