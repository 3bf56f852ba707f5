// Paged attention for a decode batch whose sequences begin with the same prefix (a system prompt held once in the
// prefix cache), one or several query tokens per sequence.  The reference has no counterpart: its decode attention
// (nano-vllm-java/src/main/java/com/igormaznitsa/nanollvm/layers/Attention.java:308-396) walks every key of every
// sequence, shared or not; the result here is the same.
//
// Query token t of sequence b stands at position pos = ctx_b - n_b + (t - cu_b) and sees the keys j <= pos (and
// j > pos - window).  Key j lives in prefix page prefix_blocks[j / bs] while j < prefix_len, else in
// block_tables[b][j / bs].  A row that sees no key gives zeros.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <string>
#include <tuple>

#include "common.cuh"
#include "launch.h"
#include "tma_host.h"

namespace {

using bf16 = __nv_bfloat16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxHd = 512;

// Device view of one call.
struct SpArgs {
  const bf16* q;
  long q_tok, q_head;  // strides, elements
  bf16* out;
  long o_tok, o_head;
  const int* prefix_blocks;
  int n_prefix_blocks;
  int prefix_len_host;
  const int* prefix_len_dev;  // overrides prefix_len_host when set (read on the device: graph replays may change it)
  const int* block_tables;
  long bt_stride;
  int bt_width;
  const int* ctx_lens;
  const int* cu_q;  // null: one token per sequence
  int B, T, nq, nkv, hd, block_size, num_blocks, max_q, max_len;
  float scale, softcap;
  int window;
  int* err;

  NV_DEVICE int prefix_len() const { return prefix_len_dev != nullptr ? *prefix_len_dev : prefix_len_host; }
  NV_DEVICE bool prefix_ok(int P) const { return P >= 0 && (long)P <= (long)n_prefix_blocks * block_size; }
  // First and one-past-last query token of sequence b; an end before the first when cu_q or max_q do not fit.
  NV_DEVICE int2 tokens(int b) const {
    if (cu_q == nullptr) return make_int2(b, b + 1);
    const int a = cu_q[b], e = cu_q[b + 1];
    return a < 0 || e > T || e < a || e - a > max_q ? make_int2(0, -1) : make_int2(a, e);
  }
  // Whether the block tables cover the keys of sequence b.
  NV_DEVICE bool ctx_ok(int ctx, int P) const {
    return ctx >= 0 && ctx <= max_len && (ctx <= P || (long)ctx <= (long)bt_width * block_size);
  }
};

// cap * tanh(x / cap); tanh from the exponential (the approximate tanh instruction is off by up to 2^-11, which an
// exponential of the score turns into percents)
__device__ __forceinline__ float sp_cap(float x, float cap) {
  if (cap <= 0.f) return x;
  const float e = exp2f(2.f * kLog2e / cap * x);
  return cap * (1.f - 2.f / (e + 1.f));
}

// Sequence of query token t: the last b with cu_q[b] <= t (the caller checks t < cu_q[b + 1]).
__device__ __forceinline__ int seq_of(const int* cu_q, int B, int t) {
  int lo = 0, hi = B;  // cu_q[lo] <= t < cu_q[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_q[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One warp per (query token, head), online softmax over the keys.
__global__ void __launch_bounds__(128) sp_generic_kernel(SpArgs a, const bf16* __restrict__ kc,
                                                         const bf16* __restrict__ vc) {
  nvb::pdl_wait();
  nvb::pdl_trigger();
  const long wg = ((long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (wg >= (long)a.T * a.nq) return;
  const int t = (int)(wg / a.nq), h = (int)(wg % a.nq);
  const int P = a.prefix_len();
  const int b = a.cu_q == nullptr ? t : seq_of(a.cu_q, a.B, t);
  const int2 tk = a.tokens(b);
  const int ctx = a.ctx_lens[b];
  if (!a.prefix_ok(P) || tk.y < tk.x || !a.ctx_ok(ctx, P)) {
    if (lane == 0) nvb::record_error(a.err, nvb::kErrBadArgument);
    return;
  }
  if (t < tk.x || t >= tk.y) return;  // a row behind the last sequence
  const int pos = ctx - (tk.y - tk.x) + (t - tk.x);
  const int kvh = h / (a.nq / a.nkv);
  const int key_begin = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  constexpr int PER = kMaxHd / 32;
  float qv[PER], acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int d = lane + 32 * i;
    qv[i] = d < a.hd ? __bfloat162float(a.q[t * a.q_tok + h * a.q_head + d]) : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int key = key_begin; key <= pos; ++key) {
    const int pg = key / a.block_size;
    const int blk = key < P ? a.prefix_blocks[pg] : a.block_tables[b * a.bt_stride + pg];
    if (blk < 0 || blk >= a.num_blocks) {
      if (lane == 0) nvb::record_error(a.err, nvb::kErrBadArgument);
      return;
    }
    const long off = (((long)blk * a.nkv + kvh) * a.block_size + key % a.block_size) * a.hd;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < a.hd) s += qv[i] * __bfloat162float(kc[off + lane + 32 * i]);
    const float x = sp_cap(nvb::warp_sum(s) * a.scale, a.softcap) * kLog2e;
    const float nm = fmaxf(m, x);
    const float corr = nm == -INFINITY ? 1.f : exp2f(m - nm), p = nm == -INFINITY ? 0.f : exp2f(x - nm);
    l = l * corr + p;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane + 32 * i < a.hd) acc[i] = acc[i] * corr + p * __bfloat162float(vc[off + lane + 32 * i]);
    m = nm;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane + 32 * i < a.hd) a.out[t * a.o_tok + h * a.o_head + lane + 32 * i] = __float2bfloat16(acc[i] * inv);
}

void check_i32(const at::Tensor& t, const at::Tensor& like, int64_t dim, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim && t.device() == like.device() &&
                  (t.size(-1) <= 1 || t.stride(-1) == 1),
              std::string(name) + " must be int32 on the device of q, contiguous along the last of " +
                  std::to_string(dim) + " dimension(s)");
}

}  // namespace

// q [T, nq, hd] bf16; caches [num_blocks, nkv, block, hd]; returns (out, launches).  ``prefix_len_dev`` (int32, one
// element) replaces ``prefix_len`` when given.
std::tuple<at::Tensor, int64_t> shared_prefix_attention_cuda(
    at::Tensor q, at::Tensor k_cache, at::Tensor v_cache, at::Tensor prefix_blocks, int64_t prefix_len,
    c10::optional<at::Tensor> prefix_len_dev, at::Tensor block_tables, at::Tensor ctx_lens, double scale,
    double softcap, int64_t window, c10::optional<at::Tensor> cu_q, int64_t max_q, int64_t max_len,
    c10::optional<at::Tensor> out_opt, at::Tensor err) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 3, "q must be bf16 [T, nq, hd]");
  const int64_t T = q.size(0), nq = q.size(1), hd = q.size(2);
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(),
              "caches must both be [num_blocks, nkv, block, hd]");
  for (const auto* c : {&k_cache, &v_cache})
    TORCH_CHECK(c->device() == q.device() && c->scalar_type() == at::kBFloat16 && c->is_contiguous() &&
                    (reinterpret_cast<uintptr_t>(c->data_ptr()) & 15) == 0,
                "caches must be contiguous, 16-byte aligned bf16 on the device of q");
  const int64_t NB = k_cache.size(0), nkv = k_cache.size(1), bs = k_cache.size(2), B = ctx_lens.numel();
  TORCH_CHECK(k_cache.size(3) == hd, "q and the caches differ in head dim");
  TORCH_CHECK(nkv > 0 && nq > 0 && nq % nkv == 0, "query heads must be a multiple of the KV heads");
  TORCH_CHECK(bs > 0 && bs % 64 == 0, "block size must be a multiple of 64");
  TORCH_CHECK(hd >= 8 && hd <= kMaxHd && hd % 8 == 0, "head dim must be a multiple of 8 up to 512");
  check_i32(prefix_blocks, q, 1, "prefix_blocks");
  check_i32(block_tables, q, 2, "block_tables");
  check_i32(ctx_lens, q, 1, "ctx_lens");
  TORCH_CHECK(block_tables.size(0) == B, "block_tables must have one row per sequence");
  if (prefix_len_dev.has_value()) {
    TORCH_CHECK(prefix_len_dev->scalar_type() == at::kInt && prefix_len_dev->numel() == 1 &&
                    prefix_len_dev->device() == q.device(),
                "prefix_len must be an int or one int32 on the device of q");
  } else {
    TORCH_CHECK(prefix_len >= 0 && prefix_len <= prefix_blocks.numel() * bs,
                "prefix_len must lie between 0 and the keys of prefix_blocks");
  }
  if (cu_q.has_value()) {
    check_i32(*cu_q, q, 1, "cu_q");
    TORCH_CHECK(cu_q->numel() == B + 1, "cu_q must have one entry more than there are sequences");
  } else {
    TORCH_CHECK(T == B, "without cu_q there is one query token per sequence");
  }
  TORCH_CHECK(max_q >= 1 && max_len >= 0 && window >= 0 && softcap >= 0.0, "max_q must be at least 1; max_len, window "
              "and softcap not negative");
  TORCH_CHECK(std::isfinite(scale) && std::isfinite(softcap), "scale and softcap must be finite");
  TORCH_CHECK(max_len < (int64_t(1) << 30) && T * nq < (int64_t(1) << 30) && window < (int64_t(1) << 30),
              "more keys or query rows than the kernels index");
  for (int64_t i = 0; i < 2; ++i)
    TORCH_CHECK(q.stride(i) % 8 == 0, "q rows must start on 16-byte boundaries");
  TORCH_CHECK(T == 0 || (q.stride(2) == 1 && (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0),
              "q rows must be contiguous and start on 16-byte boundaries");
  const c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out;
  if (out_opt.has_value()) {
    out = *out_opt;
    TORCH_CHECK(out.device() == q.device() && out.scalar_type() == at::kBFloat16 && out.sizes() == q.sizes(),
                "out must be bf16 of the shape and device of q");
    TORCH_CHECK(T == 0 || (out.stride(2) == 1 && out.stride(0) % 8 == 0 && out.stride(1) % 8 == 0 &&
                           (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15) == 0),
                "out rows must be contiguous and start on 16-byte boundaries");
  } else {
    out = at::empty({T, nq, hd}, q.options());
  }
  if (T == 0 || B == 0) return {out, 0};
  TORCH_CHECK(NB > 0, "the caches hold no pages");

  SpArgs a{};
  a.q = reinterpret_cast<const bf16*>(q.data_ptr());
  a.q_tok = q.stride(0), a.q_head = q.stride(1);
  a.out = reinterpret_cast<bf16*>(out.data_ptr());
  a.o_tok = out.stride(0), a.o_head = out.stride(1);
  a.prefix_blocks = prefix_blocks.data_ptr<int>();
  a.n_prefix_blocks = (int)prefix_blocks.numel();
  a.prefix_len_host = (int)prefix_len;
  a.prefix_len_dev = prefix_len_dev.has_value() ? prefix_len_dev->data_ptr<int>() : nullptr;
  a.block_tables = block_tables.data_ptr<int>();
  a.bt_stride = block_tables.stride(0);
  a.bt_width = (int)block_tables.size(1);
  a.ctx_lens = ctx_lens.data_ptr<int>();
  a.cu_q = cu_q.has_value() ? cu_q->data_ptr<int>() : nullptr;
  a.B = (int)B, a.T = (int)T, a.nq = (int)nq, a.nkv = (int)nkv, a.hd = (int)hd;
  a.block_size = (int)bs, a.num_blocks = (int)NB, a.max_q = (int)max_q, a.max_len = (int)max_len;
  a.scale = (float)scale, a.softcap = (float)softcap, a.window = (int)window;
  a.err = err.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  const long warps = (long)T * nq;
  C10_CUDA_CHECK(nvb::launch(sp_generic_kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, stream, a,
                             reinterpret_cast<const bf16*>(k_cache.data_ptr()),
                             reinterpret_cast<const bf16*>(v_cache.data_ptr())));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {out, 1};
}
