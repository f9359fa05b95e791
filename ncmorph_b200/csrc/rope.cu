// Rotary positions on rows of heads at their own positions (ncm_rope_bf16):
//   (a, b) -> (a c - b s, b c + a s)
// for the pairs (x[i], x[i + r/2]) or (x[2i], x[2i + 1]), i < r/2, of every
// head's first r columns, c and s row positions[t] of the tables. Products and
// sums are separate f32 operations (no contraction), rounded once to bf16.
//
// Bound: memory. A rotated element is read and written once (4 bytes); the
// table rows add 4 r bytes per token and are shared by its heads through L1.
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
  uint32_t magic_row, magic_head;
  float sign;  // -1 for the inverse rotation
  int* err;
};

constexpr int kRopeThreads = 256;

__device__ __forceinline__ uint4 load16(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float ra = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = ra;
}

// A unit is what one thread moves at a time. VEC: 16-byte pieces (half layout:
// the two pieces of eight pairs; interleaved: one piece of four pairs; behind
// the rotated columns: one piece copied); otherwise one pair, or one column copied.
template <bool VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRopeThreads) rope_rows_kernel(const RopeArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  const long long t0 = static_cast<long long>(blockIdx.x) * a.tokens;
  const int n = static_cast<int>(min(static_cast<long long>(a.tokens), a.T - t0)) * a.row_units;
#pragma unroll 2
  for (int u = threadIdx.x; u < n; u += kRopeThreads) {
    const int tl = a.tokens == 1 ? 0 : a.row_units == 1 ? u : static_cast<int>(__umulhi(u, a.magic_row));
    const int ur = u - tl * a.row_units;
    const int head = a.head_units == 1 ? ur : static_cast<int>(__umulhi(ur, a.magic_head));
    const int w = ur - head * a.head_units;
    const long long t = t0 + tl;
    const int pos = __ldg(a.positions + t);
    if (pos < 0 || pos >= a.table_rows) {
      if (ur == 0) atomicOr(a.err, kErrBadIndex);
      continue;
    }
    const uint16_t* xr = a.x + t * a.x_stride + static_cast<long long>(head) * a.head_dim;
    uint16_t* yr = a.y + t * a.y_stride + static_cast<long long>(head) * a.head_dim;
    const float* cr = a.cos_t + static_cast<long long>(pos) * a.rotary;
    const float* sr = a.sin_t + static_cast<long long>(pos) * a.rotary;
    if (w >= a.rot_units) {
      if constexpr (VEC) {
        const int i = a.rotary + (w - a.rot_units) * 8;
        *reinterpret_cast<uint4*>(yr + i) = load16(xr + i);
      } else {
        const int i = a.rotary + (w - a.rot_units);
        yr[i] = xr[i];
      }
    } else if constexpr (!VEC) {
      const int i = INTERLEAVED ? 2 * w : w, j = INTERLEAVED ? 2 * w + 1 : w + a.half;
      float p = bf16_to_f32(xr[i]), q = bf16_to_f32(xr[j]);
      rotate(p, q, cr[w], a.sign * sr[w]);
      yr[i] = f32_to_bf16(p);
      yr[j] = f32_to_bf16(q);
    } else if constexpr (INTERLEAVED) {
      const uint4 v = load16(xr + 8 * w);
      uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float p = bf16lo(e[k]), q = bf16hi(e[k]);
        rotate(p, q, cr[4 * w + k], a.sign * sr[4 * w + k]);
        e[k] = pack_bf16x2(p, q);
      }
      *reinterpret_cast<uint4*>(yr + 8 * w) = make_uint4(e[0], e[1], e[2], e[3]);
    } else {
      const uint4 v = load16(xr + 8 * w), z = load16(xr + a.half + 8 * w);
      uint32_t e[4] = {v.x, v.y, v.z, v.w}, f[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float p0 = bf16lo(e[k]), q0 = bf16lo(f[k]), p1 = bf16hi(e[k]), q1 = bf16hi(f[k]);
        rotate(p0, q0, cr[8 * w + 2 * k], a.sign * sr[8 * w + 2 * k]);
        rotate(p1, q1, cr[8 * w + 2 * k + 1], a.sign * sr[8 * w + 2 * k + 1]);
        e[k] = pack_bf16x2(p0, p1);
        f[k] = pack_bf16x2(q0, q1);
      }
      *reinterpret_cast<uint4*>(yr + 8 * w) = make_uint4(e[0], e[1], e[2], e[3]);
      *reinterpret_cast<uint4*>(yr + a.half + 8 * w) = make_uint4(f[0], f[1], f[2], f[3]);
    }
  }
}

uint32_t magic_of(int d) { return static_cast<uint32_t>((0x100000000ull + d - 1) / d); }

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
  const bool in_place = x == y && x_stride == y_stride;
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
  const bool vec = aligned_to(x, 16) && aligned_to(y, 16) && x_stride % 8 == 0 && y_stride % 8 == 0 &&
                   head_dim % 8 == 0 && (interleaved ? rotary_dim : a.half) % 8 == 0;
  const int copied = in_place ? 0 : head_dim - rotary_dim;
  a.rot_units = vec ? (interleaved ? rotary_dim / 8 : a.half / 8) : a.half;
  a.head_units = a.rot_units + (vec ? copied / 8 : copied);
  a.row_units = heads * a.head_units;
  a.tokens = std::max(1, 2 * kRopeThreads / a.row_units);
  a.magic_row = magic_of(a.row_units);
  a.magic_head = magic_of(a.head_units);
  auto kernel = vec ? (interleaved ? rope_rows_kernel<true, true> : rope_rows_kernel<true, false>)
                    : (interleaved ? rope_rows_kernel<false, true> : rope_rows_kernel<false, false>);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Launch _launch(ctx, KID_DECODER_ELEMENTWISE, st);
  NCM_CUDA_TRY(launch_pdl(kernel, dim3(ceil_div(T, a.tokens)), dim3(kRopeThreads), 0, st, 1, a));
  return NCM_OK;
}
