// Rules on next-token logits (ncm_logits_process): repetition, frequency and
// presence penalties, biases and grammar masks, in one pass over the logits.
//
// A block owns a slice of one row's vocabulary, eight or sixteen tokens a thread. It
// loads its logits into registers first, and while they arrive counts the
// slice's tokens of the row's history in shared memory (bit 31: seen in the
// prompt; the rest: times produced; integer atomics, so the order does not
// matter) and finds the first of its bias entries for each token. Then it
// changes and writes. Tokens with a bias are written again, by the thread that
// holds their first entry, so that no thread waits for one token's bias after
// another's. What a block waits for is asked for together: the row's numbers, then
// the first eight tokens of the history and the first bias entry of every thread.
// Everything is f32, in separate operations in the documented order.
//
// Bound: memory, each logit read and written once; the history is read once per
// slice (from L2 after the first). 512 bf16 rows of 16384 with 4000 tokens, 300 biases
// and a mask each: 29 us, 2.1 TB/s moved, 0.32 of a copy: a block waits for its lists,
// counts, then writes, one after another with four barriers between, so half of the issue
// slots stay empty (27 us without the atomics); 64 KB of counts and entries and 40 registers
// x 512 threads hold an SM at three blocks, and 1024 blocks are 2.3 waves. 4 f32 rows of
// 128256: 4.8 us.
#include <algorithm>

#include "internal.h"
#include "ptx.cuh"

namespace ncm {
namespace {

constexpr int kMaxThreads = 512;
constexpr int64_t kMaxEntries = 1 << 30;  // of a list: a place plus a block's stride stays in 32 bits
constexpr uint32_t kInPrompt = 0x80000000u;
// A token's bias entries: 0 none; otherwise 2^31 - 1 minus the first one's place
// (larger is earlier), and this bit where there are more.
constexpr uint32_t kRepeated = 0x80000000u;
constexpr uint32_t kFirstEntry = 0x7FFFFFFFu;

struct LogitArgs {
  const void* in;
  void* out;
  long long in_stride, out_stride, vocab;
  ncm_logit_rules_t r;
  int* err;
};

// [lo, hi) of row r in an array of `total`; an empty range (and the error bit) where the bounds are not.
__device__ __forceinline__ void row_range(const int32_t* start, long long total, int r, int* lo, int* hi, int* err) {
  *lo = __ldg(start + r);
  *hi = __ldg(start + r + 1);
  if (*lo < 0 || *hi < *lo || *hi > total) {
    if (threadIdx.x == 0) atomicOr(err, kErrBadIndex);
    *lo = *hi = 0;
  }
}

__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = static_cast<uint16_t>(pack_rn_bf16x2(v, 0.f)); }

// Eight neighbouring logits from / to a row; `left` of them exist. VEC: the row is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int left, float (&x)[8]) {
  if (VEC && left >= 8) {
    *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
    *reinterpret_cast<float4*>(x + 4) = *reinterpret_cast<const float4*>(p + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < left ? p[i] : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t* p, int left, float (&x)[8]) {
  if (VEC && left >= 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16lo(e[i]);
      x[2 * i + 1] = bf16hi(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < left ? bf16_to_f32(p[i]) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(float* p, int left, const float (&x)[8]) {
  if (VEC && left >= 8) {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(x);
    *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(x + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = x[i];
  }
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, int left, const float (&x)[8]) {
  if (VEC && left >= 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_rn_bf16x2(x[0], x[1]), pack_rn_bf16x2(x[2], x[3]),
                                              pack_rn_bf16x2(x[4], x[5]), pack_rn_bf16x2(x[6], x[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = static_cast<uint16_t>(pack_rn_bf16x2(x[i], 0.f));
  }
}

// GROUPS of eight neighbouring tokens a thread.
template <typename TI, typename TO, bool VEC, int GROUPS>
__global__ void __launch_bounds__(kMaxThreads, 3) logits_kernel(const LogitArgs a) {
  extern __shared__ __align__(16) uint32_t sh[];
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.y, threads = blockDim.x, slice = threads * 8 * GROUPS;
  const long long v0 = static_cast<long long>(blockIdx.x) * slice;
  const int n = static_cast<int>(min(static_cast<long long>(slice), a.vocab - v0));
  const TI* in = static_cast<const TI*>(a.in) + r * a.in_stride + v0;
  TO* out = static_cast<TO*>(a.out) + r * a.out_stride + v0;
  float x[GROUPS][8];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int i = (g * threads + threadIdx.x) * 8;
    load8<VEC>(in + i, n - i, x[g]);
  }
  const ncm_logit_rules_t& R = a.r;
  const bool history = R.tokens != nullptr, biased = R.bias != nullptr;
  uint32_t* count = sh;
  uint32_t* entry = sh + slice;  // (with biases; the counts' place then exists without a history, too)
  int t_lo = 0, t_hi = 0, b_lo = 0, b_hi = 0;
  if (history) {
    row_range(R.token_start, R.num_tokens, r, &t_lo, &t_hi, a.err);
    for (int i = threadIdx.x; i < slice / 4; i += threads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (biased) {
    row_range(R.bias_start, R.num_bias, r, &b_lo, &b_hi, a.err);
    for (int i = threadIdx.x; i < slice / 4; i += threads) reinterpret_cast<uint4*>(entry)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  // (everything that is one load away is asked for before the first wait)
  const int prompt = history && R.prompt_lens != nullptr ? __ldg(R.prompt_lens + r) : 0;
  const float rep = R.repetition != nullptr ? __ldg(R.repetition + r) : 1.f;
  const float freq = R.frequency != nullptr ? __ldg(R.frequency + r) : 0.f;
  const float pres = R.presence != nullptr ? __ldg(R.presence + r) : 0.f;
  const uint32_t* mask = nullptr;
  uint32_t bits[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) bits[g] = 0xFFu;
  if (R.allowed != nullptr) {
    const int m = R.allowed_rows != nullptr ? __ldg(R.allowed_rows + r) : r;
    if (m >= 0 && m < R.allowed_count) {
      mask = R.allowed + m * R.allowed_stride + (v0 >> 5);
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        const int i = (g * threads + threadIdx.x) * 8;
        if (i < n) bits[g] = __ldg(mask + (i >> 5)) >> (i & 31);
      }
    } else if (m != -1 && threadIdx.x == 0) {
      atomicOr(a.err, kErrBadIndex);
    }
  }
  // (the first tokens and the first bias entry of this thread, ahead of their use)
  constexpr int AHEAD = 8;
  int ahead[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = t_lo + k * threads + threadIdx.x;
    ahead[k] = i < t_hi ? __ldg(R.tokens + i) : 0;
  }
  const int my = b_lo + threadIdx.x;
  const unsigned my_id = my < b_hi ? static_cast<unsigned>(__ldg(R.bias_ids + my)) : 0u;
  const float my_bias = my < b_hi ? __ldg(R.bias + my) : 0.f;
  __syncthreads();
  const unsigned first = static_cast<unsigned>(v0), un = static_cast<unsigned>(n);
  const int t_mid = t_lo + min(max(prompt, 0), t_hi - t_lo);
  bool bad = false;
  auto note = [&](int i, int token) {
    const unsigned id = static_cast<unsigned>(token), j = id - first;
    if (j < un) {
      if (i < t_mid)
        atomicOr(count + j, kInPrompt);
      else
        atomicAdd(count + j, 1u);
    }
    bad |= id >= static_cast<unsigned>(a.vocab);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = t_lo + k * threads + threadIdx.x;
    if (i < t_hi) note(i, ahead[k]);
  }
#pragma unroll 4
  for (int i = t_lo + AHEAD * threads + threadIdx.x; i < t_hi; i += threads) note(i, __ldg(R.tokens + i));
  auto id_of = [&](int i) { return i == my ? my_id : static_cast<unsigned>(__ldg(R.bias_ids + i)); };
  // the first entry of each token, then whether there are more
  for (int i = my; i < b_hi; i += threads) {
    const unsigned id = id_of(i), j = id - first;
    if (j < un) atomicMax(entry + j, kFirstEntry - static_cast<unsigned>(i - b_lo));
    bad |= id >= static_cast<unsigned>(a.vocab);
  }
  if (bad && blockIdx.x == 0) atomicOr(a.err, kErrBadIndex);
  __syncthreads();
  if (b_hi > b_lo) {
    for (int i = my; i < b_hi; i += threads) {
      const unsigned j = id_of(i) - first;
      if (j < un && (entry[j] & ~kRepeated) != kFirstEntry - static_cast<unsigned>(i - b_lo)) atomicOr(entry + j, kRepeated);
    }
    __syncthreads();
  }
  const float inv = __frcp_rn(rep);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int i = (g * threads + threadIdx.x) * 8;
    if (i >= n) continue;
    if (history) {
      uint32_t c[8];
      *reinterpret_cast<uint4*>(c) = *reinterpret_cast<const uint4*>(count + i);
      *reinterpret_cast<uint4*>(c + 4) = *reinterpret_cast<const uint4*>(count + i + 4);
      if ((c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) != 0u) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // l / rep as l * (1 / rep): two f32 roundings instead of one, a third of the instructions
          const float y = __fmul_rn(x[g][e], x[g][e] > 0.f ? inv : rep);
          const float made = static_cast<float>(c[e] & ~kInPrompt);
          const float z = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, made)), pres);
          x[g][e] = c[e] == 0u ? x[g][e] : c[e] == kInPrompt ? y : z;
        }
      }
    }
    if (b_hi > b_lo) {  // tokens with a bias: their logits take their counts' place
      uint32_t c[8];
      *reinterpret_cast<uint4*>(c) = *reinterpret_cast<const uint4*>(entry + i);
      *reinterpret_cast<uint4*>(c + 4) = *reinterpret_cast<const uint4*>(entry + i + 4);
      if ((c[0] | c[1] | c[2] | c[3] | c[4] | c[5] | c[6] | c[7]) != 0u) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c[e] != 0u) count[i + e] = __float_as_uint(x[g][e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!((bits[g] >> e) & 1u)) x[g][e] = -__uint_as_float(0x7F800000u);
    store8<VEC>(out + i, n - i, x[g]);
  }
  if (b_hi > b_lo) {
    __syncthreads();  // (orders the stores above before the ones below, too)
    for (int i = my; i < b_hi; i += threads) {
      const unsigned id = id_of(i), j = id - first;
      if (j >= un || (entry[j] & ~kRepeated) != kFirstEntry - static_cast<unsigned>(i - b_lo)) continue;
      float y = __fadd_rn(__uint_as_float(count[j]), i == my ? my_bias : __ldg(R.bias + i));
      if (entry[j] & kRepeated)
        for (int k = i + 1; k < b_hi; ++k)
          if (static_cast<unsigned>(__ldg(R.bias_ids + k)) == id) y = __fadd_rn(y, __ldg(R.bias + k));
      if (mask != nullptr && !((__ldg(mask + (j >> 5)) >> (j & 31)) & 1u)) y = -__uint_as_float(0x7F800000u);
      store_logit(out + j, y);
    }
  }
}

}  // namespace
}  // namespace ncm

using namespace ncm;

extern "C" int ncm_logits_process(ncm_ctx_t* ctx, const void* logits, int32_t dtype, int64_t stride, void* out,
                                  int32_t out_dtype, int64_t out_stride, int64_t rows, int64_t vocab,
                                  const ncm_logit_rules_t* rules, ncm_stream_t stream) {
  DeviceGuard guard(ctx);
  if (guard.status()) return guard.status();
  if (rules == nullptr) return ncm_fail(NCM_EINVAL, "logits_process: null rules");
  if (!((dtype == NCM_DTYPE_F32 && out_dtype == NCM_DTYPE_F32) ||
        (dtype == NCM_DTYPE_BF16 && (out_dtype == NCM_DTYPE_F32 || out_dtype == NCM_DTYPE_BF16))))
    return ncm_fail(NCM_EINVAL, "logits_process: no conversion from type %d to %d", dtype, out_dtype);
  if (rows < 0 || rows > 65535 || vocab < 1 || vocab > INT32_MAX || stride < vocab || out_stride < vocab ||
      stride > INT64_MAX / 8 / (rows + 1) || out_stride > INT64_MAX / 8 / (rows + 1))
    return ncm_fail(NCM_EINVAL, "logits_process: bad shape rows=%lld vocab=%lld strides %lld, %lld", (long long)rows,
                    (long long)vocab, (long long)stride, (long long)out_stride);
  const size_t isz = dtype == NCM_DTYPE_F32 ? 4 : 2, osz = out_dtype == NCM_DTYPE_F32 ? 4 : 2;
  const ncm_logit_rules_t& r = *rules;
  if (r.tokens != nullptr && (r.token_start == nullptr || r.num_tokens < 0 || r.num_tokens > kMaxEntries))
    return ncm_fail(NCM_EINVAL, "logits_process: tokens need token_start and num_tokens (at most 2^30)");
  if (r.tokens == nullptr && (r.repetition || r.frequency || r.presence))
    return ncm_fail(NCM_EINVAL, "logits_process: penalties need tokens");
  if (r.bias != nullptr && (!r.bias_ids || !r.bias_start || r.num_bias < 0 || r.num_bias > kMaxEntries))
    return ncm_fail(NCM_EINVAL, "logits_process: bias needs bias_ids, bias_start and num_bias (at most 2^30)");
  const int64_t words = (vocab + 31) / 32;
  if (r.allowed != nullptr && (r.allowed_count < 0 || r.allowed_stride < words ||
                               r.allowed_stride > INT64_MAX / 8 / (r.allowed_count + 1)))
    return ncm_fail(NCM_EINVAL, "logits_process: masks need %lld words a row", (long long)words);
  const void* four[] = {r.tokens, r.token_start, r.prompt_lens, r.repetition, r.frequency, r.presence, r.bias_ids, r.bias,
                        r.bias_start, r.allowed, r.allowed_rows};
  for (const void* p : four)
    if (!aligned_to(p, 4)) return ncm_fail(NCM_EINVAL, "logits_process: misaligned rule array");
  if (rows == 0) return NCM_OK;
  if (!logits || !out || !aligned_to(logits, isz) || !aligned_to(out, osz))
    return ncm_fail(NCM_EINVAL, "logits_process: null or misaligned logits");
  const bool in_place = logits == out && dtype == out_dtype && (stride == out_stride || rows == 1);
  if (!in_place && ranges_overlap(logits, isz * ((rows - 1) * stride + vocab), out, osz * ((rows - 1) * out_stride + vocab)))
    return ncm_fail(NCM_EINVAL, "logits_process: logits and out overlap without being the same rows");
  LogitArgs a{logits, out, stride, out_stride, vocab, r, ctx->d_err};
  // The longest slice (its history is read the fewest times) that still gives
  // every SM four blocks; where that is not to be had, short slices of eight tokens a
  // thread, so that more threads read the history.
  int threads = kMaxThreads, groups = 2;
  while (threads > 128 && rows * ceil_div(vocab, threads * 8 * groups) < 4 * ctx->num_sms) {
    groups = 1;
    threads /= 2;
  }
  const int slice = threads * 8 * groups;
  const size_t smem = sizeof(uint32_t) * slice * (r.bias != nullptr ? 2 : r.tokens != nullptr ? 1 : 0);
  const bool vec = aligned_to(logits, 16) && aligned_to(out, 16) && stride * isz % 16 == 0 && out_stride * osz % 16 == 0;
  using Kernel = void (*)(const LogitArgs);
  static const Kernel table[3][2][2] = {
      {{logits_kernel<float, float, false, 1>, logits_kernel<float, float, false, 2>},
       {logits_kernel<float, float, true, 1>, logits_kernel<float, float, true, 2>}},
      {{logits_kernel<uint16_t, float, false, 1>, logits_kernel<uint16_t, float, false, 2>},
       {logits_kernel<uint16_t, float, true, 1>, logits_kernel<uint16_t, float, true, 2>}},
      {{logits_kernel<uint16_t, uint16_t, false, 1>, logits_kernel<uint16_t, uint16_t, false, 2>},
       {logits_kernel<uint16_t, uint16_t, true, 1>, logits_kernel<uint16_t, uint16_t, true, 2>}}};
  const int kind = dtype == NCM_DTYPE_F32 ? 0 : out_dtype == NCM_DTYPE_F32 ? 1 : 2;
  const Kernel kernel = table[kind][vec][groups - 1];
  static DeviceFlags ready[3][2][2];
  DeviceFlags& flag = ready[kind][vec][groups - 1];
  if (!flag.test(ctx->device)) {
    NCM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * sizeof(uint32_t) * kMaxThreads * 16));
    flag.set(ctx->device);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Launch _launch(ctx, KID_LOGITS, st);
  NCM_CUDA_TRY(launch_pdl(kernel, dim3(ceil_div(vocab, slice), static_cast<unsigned>(rows)), dim3(threads), smem, st, 1, a));
  return NCM_OK;
}
