// Rotary positions on rows of heads at their own positions (ncm_rope_bf16):
//   (a, b) -> (a c - b s, b c + a s)
// for the pairs (x[i], x[i + r/2]) or (x[2i], x[2i + 1]), i < r/2, of every
// head's first r columns, c and s row positions[t] of the tables. Products and
// sums are separate f32 operations (no contraction), rounded once to bf16.
//
// Bound: memory. A rotated element is read and written once (4 bytes); the
// table rows add 4 r bytes per token and are shared by its heads through L1.
// 16384 rows of 40 heads of 128 with 64 columns rotated as neighbours: 56 us, 6.06
// TB/s moved, 0.92 of a copy; as halves 62 us, 5.5 TB/s. Whole heads as halves, the decoder's
// layout: 28.2 us for 40 heads of 64, 6.1 TB/s, 0.93 of a copy, 55.9 us for 40 of 128. 48 rows
// of 40 heads of 64: 1.6 us beside its neighbours in a graph.
#include <algorithm>

#include "internal.h"
#include "ptx.cuh"

namespace ncm {
namespace {

struct RopeArgs {
  const uint16_t* x;
  uint16_t* y;
  long long x_stride, y_stride;
  const int32_t* positions;
  const float* cos_t;
  const float* sin_t;
  long long table_rows;
  long long T;
  int head_dim, rotary, half;
  int rot_units, head_units;  // units of one head: rotated ones, and all
  int row_units;              // heads * head_units
  int tokens;                 // tokens of one block
  float sign;                 // -1 for the inverse rotation
  int* err;
};

__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float ra = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = ra;
}

// A unit is what one thread moves at a time: VEC: 16-byte pieces (half layout:
// the two pieces of eight pairs; interleaved: one piece of four pairs; behind
// the rotated columns: one piece copied); otherwise one pair, or one column
// copied. A thread keeps its unit (blockIdx.y picks the part of the row) and
// walks over the block's tokens, BATCH of them loaded before the first is used: two
// are enough (us of 2, 3, 4 and 8 for the neighbours above: 56, 58, 57 and 84), at 32
// registers a thread for neighbours and 52 for halves, whose unit is two pieces. Rows pass
// the caches by (__ldcs, __stcs: 58 without).
template <bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int BATCH = 2;
  constexpr bool TWO = !INTERLEAVED || !VEC;  // a unit is two loads
  constexpr int PAIRS = VEC ? (INTERLEAVED ? 4 : 8) : 1;
  const int u = blockIdx.y * blockDim.x + threadIdx.x;
  if (u >= a.row_units) return;
  const int head = u / a.head_units, w = u - head * a.head_units;
  const bool rot = w < a.rot_units;
  int i = head * a.head_dim, step = 0;  // the unit's column, and how far its second load is
  if (rot) {
    i += VEC ? 8 * w : INTERLEAVED ? 2 * w : w;
    step = VEC || !INTERLEAVED ? a.half : 1;
  } else {
    i += a.rotary + (VEC ? 8 : 1) * (w - a.rot_units);
  }
  const long long t0 = static_cast<long long>(blockIdx.x) * a.tokens;
  const int n = static_cast<int>(min(static_cast<long long>(a.tokens), a.T - t0));
  const uint16_t* src = a.x + t0 * a.x_stride + i;
  uint16_t* dst = a.y + t0 * a.y_stride + i;
  for (int k0 = 0; k0 < n; k0 += BATCH) {
    uint4 v[BATCH], z[BATCH];
    int pos[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      if (k0 + k >= n) break;
      const uint16_t* p = src + k * a.x_stride;
      if constexpr (VEC) {
        v[k] = __ldcs(reinterpret_cast<const uint4*>(p));
        if (TWO && rot) z[k] = __ldcs(reinterpret_cast<const uint4*>(p + step));
      } else {
        v[k].x = *p;
        if (rot) z[k].x = p[step];
      }
      pos[k] = __ldg(a.positions + t0 + k0 + k);
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      if (k0 + k >= n) break;
      uint16_t* q = dst + k * a.y_stride;
      if (pos[k] < 0 || pos[k] >= a.table_rows) {
        if (w == 0) atomicOr(a.err, kErrBadIndex);
        continue;
      }
      if (rot) {
        const long long at = static_cast<long long>(pos[k]) * a.rotary + PAIRS * w;
        float c[PAIRS], s[PAIRS];
        if constexpr (VEC) {
#pragma unroll
          for (int e = 0; e < PAIRS; e += 4) {
            *reinterpret_cast<float4*>(&c[e]) = __ldg(reinterpret_cast<const float4*>(a.cos_t + at + e));
            *reinterpret_cast<float4*>(&s[e]) = __ldg(reinterpret_cast<const float4*>(a.sin_t + at + e));
          }
        } else {
          c[0] = __ldg(a.cos_t + at);
          s[0] = __ldg(a.sin_t + at);
        }
        uint32_t e[4] = {v[k].x, v[k].y, v[k].z, v[k].w}, f[4] = {z[k].x, z[k].y, z[k].z, z[k].w};
        if constexpr (!VEC) {
          float p0 = bf16lo(e[0]), q0 = bf16lo(f[0]);
          rotate(p0, q0, c[0], a.sign * s[0]);
          const uint32_t both = pack_rn_bf16x2(p0, q0);
          v[k].x = both & 0xFFFFu;
          q[step] = static_cast<uint16_t>(both >> 16);
        } else if constexpr (INTERLEAVED) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float p0 = bf16lo(e[x]), q0 = bf16hi(e[x]);
            rotate(p0, q0, c[x], a.sign * s[x]);
            e[x] = pack_rn_bf16x2(p0, q0);
          }
          v[k] = make_uint4(e[0], e[1], e[2], e[3]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            float p0 = bf16lo(e[x]), q0 = bf16lo(f[x]), p1 = bf16hi(e[x]), q1 = bf16hi(f[x]);
            rotate(p0, q0, c[2 * x], a.sign * s[2 * x]);
            rotate(p1, q1, c[2 * x + 1], a.sign * s[2 * x + 1]);
            e[x] = pack_rn_bf16x2(p0, p1);
            f[x] = pack_rn_bf16x2(q0, q1);
          }
          v[k] = make_uint4(e[0], e[1], e[2], e[3]);
          __stcs(reinterpret_cast<uint4*>(q + step), make_uint4(f[0], f[1], f[2], f[3]));
        }
      }
      if constexpr (VEC)
        __stcs(reinterpret_cast<uint4*>(q), v[k]);
      else
        *q = static_cast<uint16_t>(v[k].x);
    }
    src += BATCH * a.x_stride;
    dst += BATCH * a.y_stride;
  }
}

}  // namespace
}  // namespace ncm

using namespace ncm;

extern "C" int ncm_rope_bf16(ncm_ctx_t* ctx, const uint16_t* x, int64_t x_stride, uint16_t* y, int64_t y_stride,
                             const int32_t* positions, const float* cos_t, const float* sin_t, int64_t table_rows,
                             int64_t T, int32_t heads, int32_t head_dim, int32_t rotary_dim, int32_t interleaved,
                             int32_t inverse, ncm_stream_t stream) {
  DeviceGuard guard(ctx);
  if (guard.status()) return guard.status();
  if (T < 0 || T > INT32_MAX || heads < 1 || heads > 2048 || head_dim < 2 || head_dim > 1024 || rotary_dim < 2 ||
      rotary_dim > head_dim || rotary_dim % 2 != 0)
    return ncm_fail(NCM_EINVAL, "rope: bad shape T=%lld heads=%d head_dim=%d rotary_dim=%d", (long long)T, heads,
                    head_dim, rotary_dim);
  const int64_t width = static_cast<int64_t>(heads) * head_dim;
  if (x_stride < width || y_stride < width || x_stride > INT64_MAX / 4 / (T + 1) || y_stride > INT64_MAX / 4 / (T + 1))
    return ncm_fail(NCM_EINVAL, "rope: row strides %lld and %lld must cover %lld columns", (long long)x_stride,
                    (long long)y_stride, (long long)width);
  if (table_rows < 0 || table_rows > INT32_MAX) return ncm_fail(NCM_EINVAL, "rope: bad table_rows");
  if (T == 0) return NCM_OK;
  if (!x || !y || !positions || !cos_t || !sin_t) return ncm_fail(NCM_EINVAL, "rope: null buffer");
  if (!aligned_to(x, 2) || !aligned_to(y, 2) || !aligned_to(positions, 4) || !aligned_to(cos_t, 4) ||
      !aligned_to(sin_t, 4))
    return ncm_fail(NCM_EINVAL, "rope: misaligned buffer");
  const bool in_place = x == y && (x_stride == y_stride || T == 1);  // (a single row's stride says nothing)
  if (!in_place && ranges_overlap(x, 2 * ((T - 1) * x_stride + width), y, 2 * ((T - 1) * y_stride + width)))
    return ncm_fail(NCM_EINVAL, "rope: x and y overlap without being the same rows");
  RopeArgs a{};
  a.x = x;
  a.y = y;
  a.x_stride = x_stride;
  a.y_stride = y_stride;
  a.positions = positions;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.table_rows = table_rows;
  a.T = T;
  a.head_dim = head_dim;
  a.rotary = rotary_dim;
  a.half = rotary_dim / 2;
  a.sign = inverse ? -1.f : 1.f;
  a.err = ctx->d_err;
  const bool vec = aligned_to(x, 16) && aligned_to(y, 16) && aligned_to(cos_t, 16) && aligned_to(sin_t, 16) && x_stride % 8 == 0 && y_stride % 8 == 0 &&
                   head_dim % 8 == 0 && (interleaved ? rotary_dim : a.half) % 8 == 0;
  const int copied = in_place ? 0 : head_dim - rotary_dim;
  a.rot_units = vec ? (interleaved ? rotary_dim / 8 : a.half / 8) : a.half;
  a.head_units = a.rot_units + (vec ? copied / 8 : copied);
  a.row_units = heads * a.head_units;
  // Blocks of equal parts of a row. One token a block where there are few, so
  // that they reach every SM; up to 8 where there are enough for four blocks an SM.
  const int parts = ceil_div(a.row_units, 256);
  const int threads = ceil_div(ceil_div(a.row_units, parts), 32) * 32;
  a.tokens = static_cast<int>(std::min<int64_t>(8, std::max<int64_t>(1, T * parts / (4 * ctx->num_sms))));
  auto kernel = vec ? (interleaved ? rope_rows_kernel<true, true> : rope_rows_kernel<true, false>)
                    : (interleaved ? rope_rows_kernel<false, true> : rope_rows_kernel<false, false>);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Launch _launch(ctx, KID_DECODER_ELEMENTWISE, st);
  NCM_CUDA_TRY(launch_pdl(kernel, dim3(ceil_div(T, a.tokens), parts), dim3(threads), 0, st, 1, a));
  return NCM_OK;
}
