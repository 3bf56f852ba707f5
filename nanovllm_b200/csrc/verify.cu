// Verification of drafted tokens against the target model's probabilities, from given uniform random numbers.
// The reference has no counterpart; temperature, top-k and top-p mean what they mean for its sampler
// (nano-vllm-java/src/main/java/com/igormaznitsa/nanollvm/layers/Sampler.java:69-134).
//
// Row r of sequence b holds the target's logits for the token after ids[r].  x = softcap(logit) (NaN counts as -inf),
// w_i = exp((x_i - max x) / T) on the kept set S: the k largest logits (equal ones: lowest token first), of those the
// shortest prefix in that order whose mass reaches top_p.  p = w / Z.  The draft d = ids[r + 1] is accepted while
// u_r * q_d < p_d, q the distribution it was drawn from (q_d = 1 without one).  At the first refusal the next token is
// drawn from max(0, p - q) (without q: from p without d), else from p of the sequence's last row: the first token
// whose cumulated weight exceeds u * total, u the uniform of the last row.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <string>
#include <tuple>

#include "common.cuh"
#include "launch.h"

namespace {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 512;
constexpr double kLog2e64 = 1.4426950408889634074;
// masses are summed as integers (any order, same sum): 2^43 per unit, at most 2^20 weights of at most 1
constexpr float kUnit = 8796093022208.0f;
constexpr double kUnitInv = 1.0 / 8796093022208.0;
constexpr int kMaxVocab = 1 << 20;

struct VerifyArgs {
  const void* logits;
  long ld;
  int V, R, B, max_q;
  const int64_t* ids;
  const int* cu_q;
  const float* temps;
  const int* topk;
  const float* topp;
  const void* uniforms;
  int u64;  // uniforms are doubles
  const float* probs;
  long probs_ld;
  int D;
  float softcap;
  int64_t* tokens;
  int* counts;
  // per row: kept set as a composite key (logit order, then token), acceptance
  unsigned long long* cut;
  int* accept;
  int* err;

  NV_DEVICE double uniform(int r) const {
    return u64 ? reinterpret_cast<const double*>(uniforms)[r] : (double)reinterpret_cast<const float*>(uniforms)[r];
  }
};

template <typename T>
NV_DEVICE float raw_logit(const T* p, long i);
template <>
NV_DEVICE float raw_logit<float>(const float* p, long i) {
  const float x = p[i];
  return isnan(x) ? -INFINITY : x;
}
template <>
NV_DEVICE float raw_logit<bf16>(const bf16* p, long i) {
  const float x = __bfloat162float(p[i]);
  return isnan(x) ? -INFINITY : x;
}
NV_DEVICE uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// larger = earlier in the order "logit descending, token ascending"; -0 and +0 are one value
NV_DEVICE unsigned long long rank_key(float x, int i) {
  return ((unsigned long long)order_key(x + 0.f) << 32) | (0xffffffffu - (uint32_t)i);
}

// Weights of a row relative to its largest logit.
struct RowScale {
  float m, softcap;   // largest (uncapped) logit
  float mc;           // its capped value
  float c_hi, c_lo;   // log2(e) / T as two floats
  double m64, c64, cap64;

  NV_DEVICE RowScale(float m_, float cap, float T) : m(m_), softcap(cap) {
    c64 = kLog2e64 / (double)T;
    c_hi = (float)c64;
    c_lo = (float)(c64 - (double)c_hi);
    cap64 = cap;
    mc = capped(m);
    m64 = capped64(m);
  }
  NV_DEVICE float capped(float x) const {
    if (softcap <= 0.f) return x;
    const float e = exp2f(2.8853900817779268f / softcap * x);
    return softcap * (1.f - 2.f / (e + 1.f));
  }
  NV_DEVICE double capped64(float x) const { return softcap > 0.f ? cap64 * tanh((double)x / cap64) : (double)x; }
  NV_DEVICE float weight(float x) const {
    if (x == m) return m == -INFINITY ? 0.f : 1.f;
    const float d = capped(x) - mc;
    if (d < -1e30f) return 0.f;  // masked (the type's lowest value, -inf) or below a +inf: no product to overflow
    return exp2f(fminf(0.f, fmaf(d, c_hi, d * c_lo)));
  }
  NV_DEVICE double weight64(float x) const {
    if (x == m) return m == -INFINITY ? 0.0 : 1.0;
    const double d = capped64(x) - m64;
    return d < -1e30 ? 0.0 : exp2(d * c64);
  }
};

template <typename T>
NV_DEVICE T block_sum(T v, T* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  T r = sh[0];
  for (int i = 1; i < kThreads / 32; ++i) r += sh[i];
  return r;
}

NV_DEVICE int seq_of_row(const int* cu_q, int B, int r) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu_q[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The sequence's rows, or an empty range when cu_q or max_q do not fit.
NV_DEVICE int2 seq_rows(const VerifyArgs& a, int b) {
  const int lo = a.cu_q[b], hi = a.cu_q[b + 1];
  if (lo < 0 || hi > a.R || hi < lo || hi - lo > a.max_q) return make_int2(0, -1);
  return make_int2(lo, hi);
}
// Row of the draft distributions of the draft after target row r of sequence b.
NV_DEVICE int draft_row(const VerifyArgs& a, int b, int r, int* sh) {
  int nonempty = 0;
  for (int i = threadIdx.x; i < b; i += kThreads) nonempty += a.cu_q[i + 1] > a.cu_q[i];
  return r - block_sum(nonempty, sh);
}

// One CTA per row: the kept set and, where the row holds a draft, its acceptance.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(VerifyArgs a) {
  nvb::pdl_wait();
  nvb::pdl_trigger();
  __shared__ unsigned long long hist[256], sh_u[32];
  __shared__ float sh_f[32];
  __shared__ int sh_i[32];
  __shared__ unsigned long long sel_prefix, sel_before;
  const int r = blockIdx.x, tid = threadIdx.x, V = a.V;
  const int b = seq_of_row(a.cu_q, a.B, r);
  const int2 rows = seq_rows(a, b);
  if (r < rows.x || r >= rows.y) return;
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.ld;
  float m = -INFINITY;
  for (int i = tid; i < V; i += kThreads) m = fmaxf(m, raw_logit(x, i));
  m = nvb::warp_max(m);
  if ((tid & 31) == 0) sh_f[tid >> 5] = m;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; ++i) m = fmaxf(m, sh_f[i]);
  const RowScale rs(m, a.softcap, a.temps[b]);
  // radix select over the composite keys, 8 bits a pass: the smallest kept key when weights (1 or mass) are summed in
  // descending key order up to ``target``; of the keys >= floor_key
  auto select = [&](bool by_mass, unsigned long long target, unsigned long long floor_key) {
    unsigned long long prefix = 0, mask = 0, before = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kThreads) {
        const float xv = raw_logit(x, i);
        const unsigned long long k = rank_key(xv, i);
        if (k >= floor_key && (k & mask) == prefix)
          atomicAdd(&hist[(k >> shift) & 255], by_mass ? (unsigned long long)(rs.weight(xv) * kUnit) : 1ull);
      }
      __syncthreads();
      if (tid == 0) {
        unsigned long long cum = before;
        int bin = 255;
        for (; bin > 0; --bin) {
          if (cum + hist[bin] >= target) break;
          cum += hist[bin];
        }
        sel_prefix = prefix | ((unsigned long long)bin << shift);
        sel_before = cum;
      }
      __syncthreads();
      prefix = sel_prefix;
      before = sel_before;
      mask |= 255ull << shift;
      __syncthreads();
    }
    return prefix;
  };
  auto mass_from = [&](unsigned long long floor_key) {
    unsigned long long z = 0;
    for (int i = tid; i < V; i += kThreads) {
      const float xv = raw_logit(x, i);
      if (rank_key(xv, i) >= floor_key) z += (unsigned long long)(rs.weight(xv) * kUnit);
    }
    return block_sum(z, sh_u);
  };
  const int k = a.topk[b];
  const float top = a.topp[b];
  unsigned long long cut = 0;
  if (k > 0 && k < V) cut = select(false, (unsigned long long)k, 0);
  if (top < 1.f && m != -INFINITY) {
    const double P = (double)mass_from(cut) * (double)top;
    const unsigned long long target = P > 1.0 ? (unsigned long long)ceil(P) : 1ull;  // the first token always stays
    cut = max(cut, select(true, target, cut));
  }
  if (tid == 0) a.cut[r] = cut;
  if (r + 1 == rows.y) return;  // no draft after the last row
  const long d = a.ids[r + 1];
  const int dr = a.probs != nullptr ? draft_row(a, b, r, sh_i) : 0;
  if (a.probs != nullptr && dr >= a.D) {
    if (tid == 0) nvb::record_error(a.err, nvb::kErrBadArgument);
    if (tid == 0) a.accept[r] = 0;
    return;
  }
  const unsigned long long z = mass_from(cut);
  double w = 0.0, uq = 0.0;
  if (d >= 0 && d < V) {
    const float xv = raw_logit(x, d);
    if (rank_key(xv, (int)d) >= cut) w = rs.weight64(xv);
    uq = a.uniform(r) * (a.probs != nullptr ? (double)a.probs[dr * a.probs_ld + d] : 1.0);
  }
  double Z = (double)z * kUnitInv;
  if (fabs(uq * Z - w) <= 1e-4 * w) {  // too near for the 32-bit weights: sum the row in 64 bits
    double z64 = 0.0;
    for (int i = tid; i < V; i += kThreads) {
      const float xv = raw_logit(x, i);
      if (rank_key(xv, i) >= cut) z64 += rs.weight64(xv);
    }
    Z = block_sum(z64, reinterpret_cast<double*>(sh_u));
  }
  if (tid == 0) a.accept[r] = uq * Z < w;
}

// One CTA per sequence: the accepted drafts and the drawn token.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_draw_kernel(VerifyArgs a) {
  nvb::pdl_wait();
  nvb::pdl_trigger();
  __shared__ double sh_d[32];
  __shared__ int sh_i[32], sh_tok;
  __shared__ float sh_f[32];
  const int b = blockIdx.x, tid = threadIdx.x, V = a.V, lane = tid & 31, warp = tid >> 5;
  const int2 rows = seq_rows(a, b);
  const int n = rows.y - rows.x;
  if (n <= 0) {
    for (int j = tid; j < a.max_q; j += kThreads) a.tokens[(long)b * a.max_q + j] = -1;
    if (tid == 0) {
      a.counts[b] = 0;
      if (n < 0) nvb::record_error(a.err, nvb::kErrBadArgument);
    }
    return;
  }
  int acc = 0;
  while (acc < n - 1 && a.accept[rows.x + acc]) ++acc;
  const int r = rows.x + acc;
  const bool rejected = acc < n - 1;
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.ld;
  const unsigned long long cut = a.cut[r];
  float m = -INFINITY;
  for (int i = tid; i < V; i += kThreads) m = fmaxf(m, raw_logit(x, i));
  m = nvb::warp_max(m);
  if (lane == 0) sh_f[warp] = m;
  __syncthreads();
  for (int i = 0; i < kThreads / 32; ++i) m = fmaxf(m, sh_f[i]);
  const RowScale rs(m, a.softcap, a.temps[b]);
  auto weight = [&](int i) {
    const float xv = raw_logit(x, i);
    return rank_key(xv, i) >= cut ? rs.weight64(xv) : 0.0;
  };
  double z = 0.0;
  for (int i = tid; i < V; i += kThreads) z += weight(i);
  const double Z = block_sum(z, sh_d);
  const int dr = rejected && a.probs != nullptr ? draft_row(a, b, r, sh_i) : 0;
  const float* q = rejected && a.probs != nullptr && dr < a.D ? a.probs + dr * a.probs_ld : nullptr;
  const long drafted = rejected && a.probs == nullptr ? a.ids[r + 1] : -1;
  const int chunk = (V + kThreads - 1) / kThreads, c0 = min(V, tid * chunk), c1 = min(V, c0 + chunk);
  for (int plain = rejected ? 0 : 1; plain < 2; ++plain) {
    // plain: the probabilities themselves (also when nothing is left of p - q)
    auto left = [&](int i) {
      const double w = weight(i);
      if (plain || w == 0.0) return w;
      if (q != nullptr) return fmax(0.0, w / Z - (double)q[i]);
      return i == drafted ? 0.0 : w;
    };
    double s = 0.0;
    for (int i = c0; i < c1; ++i) s += left(i);
    double incl = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) sh_d[warp] = incl;
    if (tid == 0) sh_tok = 0x7fffffff;
    __syncthreads();
    double base = 0.0, total = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) base += sh_d[i];
      total += sh_d[i];
    }
    if (total > 0.0) {
      // below total whatever the uniform is, so some token exceeds it
      const double want = fmin(fmax(a.uniform(rows.y - 1), 0.0), 1.0 - 2.220446049250313e-16) * total;
      double c = base + incl - s;
      if (s > 0.0 && base + incl > want) {
        int tok = -1;
        for (int i = c0; i < c1; ++i) {
          const double v = left(i);
          c += v;
          if (v > 0.0) tok = i;
          if (v > 0.0 && c > want) break;
        }
        atomicMin(&sh_tok, tok);
      }
    }
    __syncthreads();
    if (total > 0.0) break;
  }
  if (tid == 0) {
    int64_t* out = a.tokens + (long)b * a.max_q;
    for (int j = 0; j < a.max_q; ++j) out[j] = j < acc ? a.ids[rows.x + j + 1] : -1;
    out[acc] = sh_tok == 0x7fffffff ? 0 : sh_tok;
    a.counts[b] = acc + 1;
  }
}

}  // namespace

// logits [R, V] bf16 or fp32; ids [R] int64; cu_q [B + 1] int32; temps / topk / topp [B]; uniforms [R] fp32 or fp64;
// probs (optional) fp32 [drafts, V].  Returns (tokens int64 [B, max_q], counts int32 [B], launches).
std::tuple<at::Tensor, at::Tensor, int64_t> verify_drafts_cuda(
    at::Tensor logits, at::Tensor ids, at::Tensor cu_q, int64_t max_q, at::Tensor temps, at::Tensor topk,
    at::Tensor topp, at::Tensor uniforms, c10::optional<at::Tensor> probs, double softcap, at::Tensor err) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 &&
                  (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat),
              "logits must be bf16 or fp32 [rows, vocabulary]");
  const int64_t R = logits.size(0), V = logits.size(1), B = cu_q.numel() - 1;
  TORCH_CHECK(V >= 1 && V <= kMaxVocab, "the vocabulary must have 1 to 1048576 tokens");
  TORCH_CHECK(R == 0 || V == 1 || logits.stride(1) == 1, "logits rows must be contiguous");
  auto vec = [&](const at::Tensor& t, at::ScalarType type, int64_t n, const char* what) {
    TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && t.numel() == n && t.is_contiguous() &&
                    t.device() == logits.device(),
                std::string(what) + " must be a contiguous vector of " + std::to_string(n) + " elements of type " +
                    c10::toString(type) + " on the device of logits");
  };
  TORCH_CHECK(cu_q.dim() == 1 && B >= 0, "cu_q must have one entry more than there are sequences");
  vec(cu_q, at::kInt, B + 1, "cu_q");
  vec(ids, at::kLong, R, "ids");
  vec(temps, at::kFloat, B, "temps");
  vec(topk, at::kInt, B, "top_ks");
  vec(topp, at::kFloat, B, "top_ps");
  vec(uniforms, uniforms.scalar_type() == at::kDouble ? at::kDouble : at::kFloat, R, "uniforms");
  TORCH_CHECK(max_q >= 1, "max_q must be at least 1");
  TORCH_CHECK(std::isfinite(softcap) && softcap >= 0.0, "softcap must be finite and not negative");
  if (probs.has_value())
    TORCH_CHECK(probs->scalar_type() == at::kFloat && probs->dim() == 2 && probs->size(1) == V &&
                    (probs->size(0) == 0 || V == 1 || probs->stride(1) == 1) && probs->device() == logits.device(),
                "draft_probs must be fp32 [drafts, vocabulary] with contiguous rows on the device of logits");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto tokens = at::empty({B, max_q}, ids.options());
  auto counts = at::empty({B}, cu_q.options());
  if (B == 0) return {tokens, counts, 0};
  auto scratch = at::empty({R * 2}, ids.options());
  VerifyArgs a{};
  a.logits = logits.data_ptr();
  a.ld = logits.stride(0);
  a.V = (int)V, a.R = (int)R, a.B = (int)B, a.max_q = (int)max_q;
  a.ids = ids.data_ptr<int64_t>();
  a.cu_q = cu_q.data_ptr<int>();
  a.temps = temps.data_ptr<float>();
  a.topk = topk.data_ptr<int>();
  a.topp = topp.data_ptr<float>();
  a.uniforms = uniforms.data_ptr();
  a.u64 = uniforms.scalar_type() == at::kDouble;
  if (probs.has_value()) {
    a.probs = probs->data_ptr<float>();
    a.probs_ld = probs->stride(0);
    a.D = (int)probs->size(0);
  }
  a.softcap = (float)softcap;
  a.tokens = tokens.data_ptr<int64_t>();
  a.counts = counts.data_ptr<int>();
  a.cut = reinterpret_cast<unsigned long long*>(scratch.data_ptr<int64_t>());
  a.accept = reinterpret_cast<int*>(scratch.data_ptr<int64_t>() + R);
  a.err = err.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool wide = logits.scalar_type() == at::kFloat;
  if (R > 0) {
    C10_CUDA_CHECK(nvb::launch(wide ? verify_rows_kernel<float> : verify_rows_kernel<bf16>, dim3((unsigned)R),
                               dim3(kThreads), 0, stream, a));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  C10_CUDA_CHECK(nvb::launch(wide ? verify_draw_kernel<float> : verify_draw_kernel<bf16>, dim3((unsigned)B),
                             dim3(kThreads), 0, stream, a));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {tokens, counts, R > 0 ? 2 : 1};
}
