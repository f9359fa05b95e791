// Rules on next-token logits (ncm_logits_process): repetition, frequency and
// presence penalties, biases and grammar masks, in one pass over the logits.
//
// A block owns a slice of one row's vocabulary. It counts the slice's tokens
// of the row's history in shared memory (bit 31: seen in the prompt; the rest:
// times produced; integer atomics, so the order does not matter), finds the
// first of its bias entries for each token, and then streams the slice: read,
// change, write. Everything is f32, in separate operations in the documented order.
//
// Bound: memory, each logit read and written once. The history is read once
// per slice (from L2 after the first).
#include <algorithm>

#include "internal.h"
#include "ptx.cuh"

namespace ncm {
namespace {

constexpr int kLogitThreads = 512;
constexpr int kSlice = 8192;  // tokens of a block: 32 KB of counts, 32 KB of bias entries
constexpr uint32_t kInPrompt = 0x80000000u;
constexpr uint32_t kNoEntry = 0xFFFFFFFFu;
constexpr uint32_t kRepeated = 0x80000000u;  // more than one bias entry of this token

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

template <typename T>
__device__ __forceinline__ float load_logit(const T* p);
template <>
__device__ __forceinline__ float load_logit(const float* p) {
  return *p;
}
template <>
__device__ __forceinline__ float load_logit(const uint16_t* p) {
  return bf16_to_f32(*p);
}
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(uint16_t* p, float v) { *p = f32_to_bf16(v); }

template <typename TI, typename TO>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const LogitArgs a) {
  extern __shared__ uint32_t sh[];
  pdl_wait();
  pdl_launch_dependents();
  const int r = blockIdx.y;
  const long long v0 = static_cast<long long>(blockIdx.x) * kSlice;
  const int n = static_cast<int>(min(static_cast<long long>(kSlice), a.vocab - v0));
  const ncm_logit_rules_t& R = a.r;
  const bool history = R.tokens != nullptr, biased = R.bias != nullptr;
  uint32_t* count = sh;
  uint32_t* entry = sh + (history ? kSlice : 0);
  int t_lo = 0, t_hi = 0, b_lo = 0, b_hi = 0;
  if (history) {
    row_range(R.token_start, R.num_tokens, r, &t_lo, &t_hi, a.err);
    for (int i = threadIdx.x; i < n; i += kLogitThreads) count[i] = 0;
  }
  if (biased) {
    row_range(R.bias_start, R.num_bias, r, &b_lo, &b_hi, a.err);
    for (int i = threadIdx.x; i < n; i += kLogitThreads) entry[i] = kNoEntry;
  }
  __syncthreads();
  const int prompt = history && R.prompt_lens != nullptr ? __ldg(R.prompt_lens + r) : 0;
  for (int i = t_lo + threadIdx.x; i < t_hi; i += kLogitThreads) {
    const int id = __ldg(R.tokens + i);
    if (id < 0 || id >= a.vocab) {
      if (blockIdx.x == 0) atomicOr(a.err, kErrBadIndex);
      continue;
    }
    const long long j = id - v0;
    if (j < 0 || j >= n) continue;
    if (i - t_lo < prompt)
      atomicOr(count + j, kInPrompt);
    else
      atomicAdd(count + j, 1u);
  }
  // the first entry of each token, and whether there are more
  for (int i = b_lo + threadIdx.x; i < b_hi; i += kLogitThreads) {
    const int id = __ldg(R.bias_ids + i);
    if (id < 0 || id >= a.vocab) {
      if (blockIdx.x == 0) atomicOr(a.err, kErrBadIndex);
      continue;
    }
    const long long j = id - v0;
    if (j >= 0 && j < n) atomicMin(entry + j, static_cast<uint32_t>(i - b_lo));
  }
  if (b_hi > b_lo) {
    __syncthreads();
    for (int i = b_lo + threadIdx.x; i < b_hi; i += kLogitThreads) {
      const long long j = __ldg(R.bias_ids + i) - v0;
      if (j >= 0 && j < n && (entry[j] & ~kRepeated) != static_cast<uint32_t>(i - b_lo)) atomicOr(entry + j, kRepeated);
    }
  }
  __syncthreads();
  const uint32_t* mask = nullptr;
  if (R.allowed != nullptr) {
    const int m = R.allowed_rows != nullptr ? __ldg(R.allowed_rows + r) : r;
    if (m >= 0 && m < R.allowed_count)
      mask = R.allowed + m * R.allowed_stride;
    else if (m != -1 && threadIdx.x == 0)
      atomicOr(a.err, kErrBadIndex);
  }
  const float rep = R.repetition != nullptr ? __ldg(R.repetition + r) : 1.f;
  const float freq = R.frequency != nullptr ? __ldg(R.frequency + r) : 0.f;
  const float pres = R.presence != nullptr ? __ldg(R.presence + r) : 0.f;
  const TI* in = static_cast<const TI*>(a.in) + r * a.in_stride + v0;
  TO* out = static_cast<TO*>(a.out) + r * a.out_stride + v0;
  for (int i = threadIdx.x; i < n; i += kLogitThreads) {
    float x = load_logit(in + i);
    const uint32_t c = history ? count[i] : 0u;
    if (c != 0u) {
      x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      const uint32_t made = c & ~kInPrompt;
      if (made != 0u) x = __fsub_rn(__fsub_rn(x, __fmul_rn(freq, static_cast<float>(made))), pres);
    }
    const uint32_t e = biased ? entry[i] : kNoEntry;
    if (e != kNoEntry) {
      const int at = b_lo + static_cast<int>(e & ~kRepeated);
      x = __fadd_rn(x, __ldg(R.bias + at));
      if (e & kRepeated)
        for (int k = at + 1; k < b_hi; ++k)
          if (__ldg(R.bias_ids + k) == v0 + i) x = __fadd_rn(x, __ldg(R.bias + k));
    }
    if (mask != nullptr && !((__ldg(mask + ((v0 + i) >> 5)) >> (i & 31)) & 1u)) x = -__uint_as_float(0x7F800000u);
    store_logit(out + i, x);
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
  if (r.tokens != nullptr && (r.token_start == nullptr || r.num_tokens < 0 || r.num_tokens > INT32_MAX))
    return ncm_fail(NCM_EINVAL, "logits_process: tokens need token_start and num_tokens");
  if (r.tokens == nullptr && (r.repetition || r.frequency || r.presence))
    return ncm_fail(NCM_EINVAL, "logits_process: penalties need tokens");
  if (r.bias != nullptr && (!r.bias_ids || !r.bias_start || r.num_bias < 0 || r.num_bias > INT32_MAX))
    return ncm_fail(NCM_EINVAL, "logits_process: bias needs bias_ids, bias_start and num_bias");
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
  const bool in_place = logits == out && dtype == out_dtype && stride == out_stride;
  if (!in_place && ranges_overlap(logits, isz * ((rows - 1) * stride + vocab), out, osz * ((rows - 1) * out_stride + vocab)))
    return ncm_fail(NCM_EINVAL, "logits_process: logits and out overlap without being the same rows");
  LogitArgs a{logits, out, stride, out_stride, vocab, r, ctx->d_err};
  const size_t smem = sizeof(uint32_t) * kSlice * ((r.tokens != nullptr) + (r.bias != nullptr));
  auto kernel = dtype == NCM_DTYPE_F32      ? logits_kernel<float, float>
                : out_dtype == NCM_DTYPE_F32 ? logits_kernel<uint16_t, float>
                                             : logits_kernel<uint16_t, uint16_t>;
  static DeviceFlags ready[3];
  DeviceFlags& flag = ready[dtype == NCM_DTYPE_F32 ? 0 : out_dtype == NCM_DTYPE_F32 ? 1 : 2];
  if (!flag.test(ctx->device)) {
    NCM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * kSlice));
    flag.set(ctx->device);
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Launch _launch(ctx, KID_LOGITS, st);
  NCM_CUDA_TRY(launch_pdl(kernel, dim3(ceil_div(vocab, kSlice), static_cast<unsigned>(rows)), dim3(kLogitThreads), smem, st, 1, a));
  return NCM_OK;
}
