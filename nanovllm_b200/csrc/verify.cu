// Verification of drafted tokens against the target model's probabilities, from given uniform random numbers.
// The reference has no counterpart; temperature, top-k and top-p mean what they mean for its sampler
// (nano-vllm-java/src/main/java/com/igormaznitsa/nanollvm/layers/Sampler.java:69-134).
//
// Row r of sequence b holds the target's logits for the token after ids[r].  x = softcap(logit) (NaN counts as -inf, and
// -inf stays -inf), w_i = exp((x_i - max x) / T) on the kept set S: the k largest logits (equal ones: lowest token first), of those the
// shortest prefix in that order whose mass reaches top_p.  p = w / Z.  The draft d = ids[r + 1] is accepted while
// u_r * q_d < p_d, q the distribution it was drawn from (q_d = 1 without one).  At the first refusal the next token is
// drawn from max(0, p - q) (without q: from p without d), else from p of the sequence's last row: the first token
// whose cumulated weight exceeds u * total, u the uniform of the last row.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>

#include <cfloat>
#include <cmath>
#include <string>
#include <tuple>

#include "common.cuh"
#include "launch.h"

namespace {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr double kLog2e64 = 1.4426950408889634074;
// masses in the radix select are integers (any order, same sum): 2^43 per unit, fewer than 2^20 weights of at most 1
constexpr float kUnit = 8796093022208.0f;
constexpr int kMaxVocab = 327680;  // 32-bit logits of a row in the shared memory of eight CTAs
constexpr int kMaxCluster = 8;
constexpr int kBins = 128;   // of 1/8 octave of weight below the row's largest; the last one holds the rest
constexpr int kList = 1024;  // tokens that a cut is found among by sorting
constexpr float kListMargin = 1.0001f;  // of sums of 32-bit weights

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
  // per row: kept set as a composite key (logit order, then token), largest logit, acceptance
  unsigned long long* cut;
  float* row_max;
  int* accept;
  int* err;

  NV_DEVICE double uniform(int r) const {
    return u64 ? reinterpret_cast<const double*>(uniforms)[r] : (double)reinterpret_cast<const float*>(uniforms)[r];
  }
};

template <typename T>
NV_DEVICE float to_float(T v);
template <>
NV_DEVICE float to_float<float>(float v) { return v; }
template <>
NV_DEVICE float to_float<bf16>(bf16 v) { return __bfloat162float(v); }
NV_DEVICE uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
NV_DEVICE float key_logit(unsigned long long k) {
  const uint32_t u = (uint32_t)(k >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
// larger = earlier in the order "logit descending, token ascending"; NaN is -inf, -0 and +0 are one value
NV_DEVICE unsigned long long rank_key(float x, int i) {
  return ((unsigned long long)order_key(fmaxf(x, -INFINITY) + 0.f) << 32) | (0xffffffffu - (uint32_t)i);
}

// 2^(d c) in 64 bits (relative error below 1e-12) for an exponent in [-1000, 0]: it is k / 256 + r, with a table of
// 2^(k / 256) and three terms of the exponential series for 2^r, |r| <= 1/512 (the fourth is 1.4e-13).
constexpr int kTable = 256;
NV_DEVICE double exp2_64(double d, double c, const double* table) {
  const double magic = 26388279066624.0;  // 1.5 * 2^44: the last bit of a sum with it is 1/256
  const double t = fma(d, c, magic);
  const double r = fma(d, c, magic - t);
  const int k = max(__double2loint(t), -1000 * kTable);
  double p = 5.550410866482158e-2;
  p = fma(p, r, 2.402265069591007e-1);
  p = fma(p, r, 6.931471805599453e-1);
  p = fma(p, r, 1.0) * table[k & (kTable - 1)];
  return __hiloint2double(__double2hiint(p) + (k >> 8) * (1 << 20), __double2loint(p));
}
NV_DEVICE void fill_table(double* table) {
  if (threadIdx.x < kTable) table[threadIdx.x] = exp2(threadIdx.x * (1.0 / kTable));
}

// Weights of a row relative to its largest logit.  ``weight`` (32 bits) takes the exponent's argument as a product with
// log2(e) / T in two floats, so that its error is the rounding of the result alone; sums of it are only used where
// 1e-6 does not matter, or are done over in 64 bits.
struct RowScale {
  float m, softcap, mc;  // largest logit, its capped value
  float c_hi, c_lo;      // log2(e) / T
  float floor64;         // logits below it weigh nothing in 64 bits (2^-1000)
  double c64, m64, cap64;  // m64: the capped largest logit

  NV_DEVICE RowScale(float m_, float cap, float T) : m(m_), softcap(cap) {
    c64 = kLog2e64 / (double)T;
    c_hi = (float)c64;
    c_lo = (float)(c64 - (double)c_hi);
    cap64 = cap;
    mc = capped(m);
    m64 = capped64(m);
    floor64 = fmaxf(softcap > 0.f ? -FLT_MAX : m - 690.f * T, -FLT_MAX);
  }
  NV_DEVICE float capped(float x) const {
    if (softcap <= 0.f) return x;
    const float e = exp2f(2.8853900817779268f / softcap * x);
    return softcap * (1.f - 2.f / (e + 1.f));
  }
  NV_DEVICE double capped64(float x) const { return softcap > 0.f ? cap64 * tanh((double)x / cap64) : (double)x; }
  NV_DEVICE bool simple() const { return softcap <= 0.f && fabsf(m) < INFINITY; }
  // log2 of the weight; hugely negative for NaN, -inf and the type's lowest value (no product to overflow)
  NV_DEVICE float log_weight_simple(float x) const {
    const float d = fmaxf(x - m, -1e30f);
    return fmaf(d, c_hi, d * c_lo);
  }
  NV_DEVICE float log_weight(float x) const {
    if (m == INFINITY) return x == m ? 0.f : -1e30f;
    if (softcap <= 0.f) return log_weight_simple(x);
    const float d = x == -INFINITY ? -1e30f : fmaxf(capped(x) - mc, -1e30f);
    return fminf(0.f, fmaf(d, c_hi, d * c_lo));
  }
  NV_DEVICE float weight(float x) const { return exp2f(log_weight(x)); }
  NV_DEVICE double weight64_simple(float x, const double* table) const {  // no soft-cap, finite m
    const double w = exp2_64((double)fmaxf(x, floor64) - m64, c64, table);
    return x >= floor64 ? w : 0.0;  // NaN, -inf: 0
  }
  NV_DEVICE double weight64(float x, const double* table) const {
    if (x == m) return m == -INFINITY ? 0.0 : 1.0;
    if (m == INFINITY || !(x >= floor64)) return 0.0;  // masked stays masked, also under a soft-cap
    if (softcap <= 0.f) return weight64_simple(x, table);
    const double d = fmin(capped64(x) - m64, 0.0);
    return d * c64 > -1000.0 ? exp2_64(d, c64, table) : 0.0;
  }
};

NV_DEVICE uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
template <typename T>
NV_DEVICE T peer_load(const T* p, uint32_t rank) {  // the same variable of another CTA of the cluster
  const uint32_t at = nvb::map_peer(nvb::smem_u32(p), rank);
  if constexpr (sizeof(T) == 8) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
    return *reinterpret_cast<T*>(&v);
  } else {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return *reinterpret_cast<T*>(&v);
  }
}

template <typename T>
NV_DEVICE T block_sum(T v, T* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  T r = sh[0];
  for (int i = 1; i < kWarps; ++i) r += sh[i];
  return r;
}
// Sum over the cluster, the same in every thread.  ``slot``: one for each call of a kernel.
template <typename T>
NV_DEVICE T cluster_sum(T v, T* sh, T* slot) {
  v = block_sum(v, sh);
  const uint32_t n = cluster_size();
  if (n == 1) return v;
  if (threadIdx.x == 0) *slot = v;
  nvb::cluster_sync();
  T r = peer_load(slot, 0);
  for (uint32_t i = 1; i < n; ++i) r += peer_load(slot, i);
  return r;
}
NV_DEVICE float cluster_max(float v, float* sh, float* slot) {
  v = nvb::warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) v = fmaxf(v, sh[i]);
  const uint32_t n = cluster_size();
  if (n == 1) return v;
  if (threadIdx.x == 0) *slot = v;
  nvb::cluster_sync();
  for (uint32_t i = 0; i < n; ++i) v = fmaxf(v, peer_load(slot, i));
  return v;
}

// Sequence of row r by a 32-way search of the warp: the last b with cu_q[b] <= r.
NV_DEVICE int seq_of_row(const int* cu_q, int B, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = B;
  while (len > 1) {
    const int step = (len + 31) / 32, at = lo + lane * step;
    const bool below = at < lo + len && cu_q[at] <= r;
    const int skip = max(0, __popc(__ballot_sync(0xffffffffu, below)) - 1) * step;
    lo += skip;
    len = min(step, len - skip);
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

// This CTA's part of a row in shared memory: tokens [lo, hi) of it, at the same offset in their 16 bytes as in global
// memory, so that whole words come by one asynchronous copy; what the first and last word hold besides is -inf.
template <typename T>
struct Slice {
  static constexpr int PER = 16 / sizeof(T);
  const T* words;  // 16-byte aligned
  int lo, hi, nw, first;  // token of word w, element e: first + w * PER + e
  bool bulk;

  template <typename F>
  NV_DEVICE void each(int w, F f) const {
    const uint4 v = reinterpret_cast<const uint4*>(words)[w];
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int j = 0; j < PER; ++j) f(to_float(e[j]), first + w * PER + j);
  }
};

NV_DEVICE int slice_tokens(int V, int n) { return ((V + n - 1) / n + 7) / 8 * 8; }

// Starts the load; ``finish_slice`` before the words are read.
template <typename T>
NV_DEVICE Slice<T> load_slice(const T* row, int V, uint8_t* buf, uint64_t* bar) {
  Slice<T> s;
  const int per = slice_tokens(V, cluster_size()), tid = threadIdx.x;
  s.lo = min(V, (int)nvb::cluster_ctarank() * per);
  s.hi = min(V, s.lo + per);
  const uintptr_t g0 = reinterpret_cast<uintptr_t>(row + s.lo), g1 = reinterpret_cast<uintptr_t>(row + s.hi);
  const int off = (int)(g0 & 15);
  s.words = reinterpret_cast<const T*>(buf);
  s.first = s.lo - off / (int)sizeof(T);
  s.nw = (off + (int)(g1 - g0) + 15) / 16;
  const uintptr_t a0 = (g0 + 15) & ~uintptr_t(15), a1 = g1 & ~uintptr_t(15);
  const bool bulk = a1 > a0;
  if (tid == 0) {
    nvb::mbar_init(bar, 1);
    nvb::fence_mbar_init();
    if (bulk) {
      const uint32_t bytes = (uint32_t)(a1 - a0);
      nvb::mbar_arrive_expect_tx(bar, bytes);
      asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                       nvb::smem_u32(buf + off + (a0 - g0))),
                   "l"(a0), "r"(bytes), "r"(nvb::smem_u32(bar))
                   : "memory");
    }
  }
  // the ends of the first and last word
  const int n_head = bulk ? (int)(a0 - g0) / (int)sizeof(T) : s.hi - s.lo;
  const int n_tail = bulk ? (int)(g1 - a1) / (int)sizeof(T) : 0;
  T* el = reinterpret_cast<T*>(buf);
  const int skip = off / (int)sizeof(T), n = s.hi - s.lo;
  if (tid < skip) el[tid] = (T)(-INFINITY);
  if (tid < n_head) el[skip + tid] = row[s.lo + tid];
  if (tid < n_tail) el[skip + n - n_tail + tid] = row[s.hi - n_tail + tid];
  for (int i = skip + n + tid; i < s.nw * Slice<T>::PER; i += kThreads) el[i] = (T)(-INFINITY);
  s.bulk = bulk;
  return s;
}
template <typename T>
NV_DEVICE void finish_slice(const Slice<T>& s, uint64_t* bar, int* err) {
  __syncthreads();
  if (s.bulk) nvb::mbar_wait(bar, 0, err, nullptr);
}

// One cluster per row: the kept set and, where the row holds a draft, its acceptance.  The row stays in the cluster's
// shared memory, every pass after the load reads it there; bound by the bytes of the logits.
//   no cut     maximum, sum of the weights
//   top_k 1    maximum, its lowest token
//   cuts       counts by 1/8 octave of weight bound where the cut falls; the tokens above that (and one bin more, so
//              that roundings of the weight do not matter) are sorted when they are few, else the tokens of the bins in
//              question go through a radix select over composite keys
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const VerifyArgs a) {
  nvb::pdl_wait();
  nvb::pdl_trigger();
  extern __shared__ __align__(128) uint8_t buf[];
  __shared__ uint64_t bar;
  __shared__ float sh_f[32], slot_f;
  __shared__ double sh_d[32], slot_d[3], table[kTable];
  __shared__ int sh_i[32];
  __shared__ unsigned long long sh_u[32], slot_u[4];
  __shared__ float slot_f3[2][2];
  __shared__ unsigned int hist[kBins], hist_all[kBins];
  __shared__ unsigned long long hist_m[2][256];
  __shared__ unsigned int hist_c[2][256];
  __shared__ unsigned long long keys[kList];
  __shared__ unsigned int n_list, slot_n;
  __shared__ int sel[4];
  __shared__ unsigned long long sel_u[2], cut_sh;
  __shared__ double z_sh;
  const int r = blockIdx.x / cluster_size(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const uint32_t rank = nvb::cluster_ctarank(), CL = cluster_size();
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.ld;
  const Slice<T> s = load_slice(x, V, buf, &bar);
  const int b = seq_of_row(a.cu_q, a.B, r);
  const int2 rows = seq_rows(a, b);
  fill_table(table);
  if (tid < kBins) hist[tid] = 0;
  if (tid == 0) n_list = 0;
  finish_slice(s, &bar, a.err);
  if (r < rows.x || r >= rows.y) return;  // the whole cluster
  float m = -INFINITY;
  for (int w = tid; w < s.nw; w += kThreads) s.each(w, [&](float v, int) { m = fmaxf(m, v); });
  m = cluster_max(m, sh_f, &slot_f);
  const RowScale rs(m, a.softcap, a.temps[b]);
  const int k = a.topk[b];
  const float top = a.topp[b];
  const bool cut_k = k > 0 && k < V, cut_p = top < 1.f;
  unsigned long long cut = 0;
  double Z = 0.0;
  if (k == 1) {
    // the lowest token among the largest logits
    unsigned long long best = 0;
    for (int w = tid; w < s.nw; w += kThreads)
      s.each(w, [&](float v, int i) {
        if (v == m) best = max(best, rank_key(v, i));
      });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh_u[warp] = best;
    __syncthreads();
    for (int i = 0; i < kWarps; ++i) best = max(best, sh_u[i]);
    if (CL > 1) {
      if (tid == 0) slot_u[0] = best;
      nvb::cluster_sync();
      for (uint32_t i = 0; i < CL; ++i) best = max(best, peer_load(&slot_u[0], i));
    }
    cut = m == -INFINITY ? 0 : best;
    Z = 1.0;
  } else {
    const bool cuts = (cut_k || cut_p) && m != -INFINITY;
    float z4[4] = {0.f, 0.f, 0.f, 0.f};
    if (!cuts && rs.simple()) {
      for (int w = tid; w < s.nw; w += kThreads) {
        int j = 0;
        s.each(w, [&](float v, int) { z4[j++ & 3] += exp2f(rs.log_weight_simple(v)); });
      }
    } else {
      const bool simple = rs.simple();
      for (int w = tid; w < s.nw; w += kThreads) {
        int j = 0;
        s.each(w, [&](float v, int) {
          const float lw = simple ? rs.log_weight_simple(v) : rs.log_weight(v);
          z4[j++ & 3] += exp2f(lw);
          if (cuts && lw > -(kBins - 1) / 8.f) atomicAdd(&hist[(int)(lw * -8.f)], 1u);
        });
      }
    }
    Z = cluster_sum((double)(z4[0] + z4[1]) + (double)(z4[2] + z4[3]), sh_d, &slot_d[0]);
    if (cuts) {
      // counts of the whole row (the sum above was a barrier of the cluster, or of the only CTA)
      if (tid < kBins - 1) {
        unsigned int n = 0;
        for (uint32_t i = 0; i < CL; ++i) n += CL > 1 ? peer_load(&hist[tid], i) : hist[tid];
        hist_all[tid] = n;
      }
      __syncthreads();
      if (warp == 0) {
        // lane: 4 bins.  Counts, and the lowest, middle and highest mass that they allow, from the largest weights on
        unsigned int cnt = 0;
        float low = 0.f, mid = 0.f, high = 0.f;
        unsigned int c4[4];
        float l4[4], m4[4], h4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int bin = lane * 4 + j;
          const unsigned int n = bin < kBins - 1 ? hist_all[bin] : 0u;
          c4[j] = cnt += n;
          l4[j] = low += n * exp2f((bin + 1.01f) * -0.125f);
          m4[j] = mid += n * exp2f((bin + 0.5f) * -0.125f);
          h4[j] = high += n * exp2f((bin - 0.01f) * -0.125f);
        }
        unsigned int ci = cnt;
        float li = low, mi = mid, hi = high;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned int cu = __shfl_up_sync(0xffffffffu, ci, o);
          const float lu = __shfl_up_sync(0xffffffffu, li, o), mu = __shfl_up_sync(0xffffffffu, mi, o);
          const float hu = __shfl_up_sync(0xffffffffu, hi, o);
          if (lane >= o) ci += cu, li += lu, mi += mu, hi += hu;
        }
        const float want = (float)((double)top * Z), likely = 0.5f * (want + (float)Z);
        // first bin that certainly / probably / possibly reaches the target, and the last one that the list holds
        int sure_k = kBins - 1, sure_p = kBins - 1, prob_p = kBins - 2, may_p = kBins - 1, fit = -1;
#pragma unroll
        for (int j = 3; j >= 0; --j) {
          const int bin = lane * 4 + j;
          if (bin >= kBins - 1) continue;
          if (ci - cnt + c4[j] >= (unsigned int)k) sure_k = bin;
          if (li - low + l4[j] >= want * kListMargin) sure_p = bin;
          if (mi - mid + m4[j] >= likely) prob_p = bin;
          if (hi - high + h4[j] >= want / kListMargin) may_p = bin;
          if (ci - cnt + c4[j] <= (unsigned int)kList) fit = max(fit, bin);
        }
        sure_k = __reduce_min_sync(0xffffffffu, sure_k);
        sure_p = __reduce_min_sync(0xffffffffu, sure_p);
        prob_p = __reduce_min_sync(0xffffffffu, prob_p);
        may_p = __reduce_min_sync(0xffffffffu, may_p);
        fit = __reduce_max_sync(0xffffffffu, fit);
        if (lane == 0) {
          sel[0] = sure_k;
          sel[1] = sure_p;
          sel[2] = may_p;
          // one bin more than the one that holds the cut; a list that turns out short of the mass is given up again
          sel[3] = cut_k ? (sure_k + 1 <= fit ? sure_k + 1 : -1) : min(prob_p + 1, fit);
        }
      }
      __syncthreads();
      const int last_bin = sel[3];
      bool listed = last_bin >= 0;
      if (listed) {
        // ------------------------------------------------ few tokens: collect, sort, walk
        for (int w = tid; w < s.nw; w += kThreads)
          s.each(w, [&](float v, int i) {
            const float lw = rs.log_weight(v);
            if (lw > -(kBins - 1) / 8.f && (int)(lw * -8.f) <= last_bin)
              keys[atomicAdd(&n_list, 1u)] = rank_key(v, i);
          });
        __syncthreads();
        const unsigned int mine = n_list;
        if (CL > 1) {
          nvb::cluster_sync();
          if (rank == 0) {  // gather behind the own ones
            unsigned int at = mine;
            for (uint32_t q = 1; q < CL; ++q) {
              const unsigned int n = peer_load(&n_list, q);
              for (unsigned int i = tid; i < n; i += kThreads) keys[at + i] = peer_load(&keys[i], q);
              at += n;
            }
            if (tid == 0) slot_n = at;
          }
        } else if (tid == 0) {
          slot_n = mine;
        }
        __syncthreads();
        if (rank == 0) {
          const int n = (int)slot_n;
          int n2 = 32;
          while (n2 < n) n2 *= 2;
          for (int i = n + tid; i < n2; i += kThreads) keys[i] = 0;
          __syncthreads();
          for (int size = 2; size <= n2; size *= 2)
            for (int d = size / 2; d > 0; d /= 2) {
              for (int i = tid; i < n2 / 2; i += kThreads) {
                const int lo = 2 * i - (i & (d - 1)), hi = lo + d;
                const bool down = (lo & size) == 0;
                const unsigned long long p = keys[lo], q = keys[hi];
                if ((p < q) == down) {
                  keys[lo] = q;
                  keys[hi] = p;
                }
              }
              __syncthreads();
            }
          // weights in order, two tokens per thread, and the sums before each
          const int nk = cut_k ? min(k, n) : n;
          double w2[2], sum = 0.0;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int i = tid * 2 + j;
            w2[j] = i < nk ? rs.weight64(key_logit(keys[i]), table) : 0.0;
            sum += w2[j];
          }
          double incl = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
          }
          if (lane == 31) sh_d[warp] = incl;
          __syncthreads();
          double base = 0.0, all = 0.0;
          for (int i = 0; i < kWarps; ++i) {
            if (i < warp) base += sh_d[i];
            all += sh_d[i];
          }
          const double want = cut_p ? (double)top * (cut_k ? all : Z) : 4.0 * kMaxVocab;
          listed = cut_k || all >= want;  // with a token of each bin behind the cut's, roundings of the weights included
          double before = base + incl - sum, kept = 0.0;
          int last = -1;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int i = tid * 2 + j;
            if (i < nk && (i == 0 || before < want)) {
              last = i;
              kept += w2[j];
            }
            before += w2[j];
          }
          last = __reduce_max_sync(0xffffffffu, last);
          if (lane == 0) sh_i[warp] = last;
          kept = block_sum(kept, sh_d);
          for (int i = 0; i < kWarps; ++i) last = max(last, sh_i[i]);
          if (tid == 0) {
            cut_sh = keys[last];
            z_sh = kept;
          }
          __syncthreads();
          if (listed) {
            cut = cut_sh;
            Z = z_sh;
          }
          if (tid == 0) sel_u[0] = listed;
          __syncthreads();
        }
        if (CL > 1 && !cut_k) {
          nvb::cluster_sync();
          listed = peer_load(&sel_u[0], 0) != 0;
          nvb::cluster_sync();
        }
      }
      if (!listed) {
        // ------------------------------------------------ many: radix select over the tokens whose logits lie in the
        // range of those in the bins in question
        auto bin_of = [&](float v) {
          const float lw = rs.log_weight(v);
          return lw > -(kBins - 1) / 8.f ? (int)(lw * -8.f) : kBins - 1;
        };
        // sum of 1 or of the masses over f(logit, token)
        auto total_of = [&](bool by_mass, unsigned long long* slot, auto f) {
          unsigned long long n = 0;
          for (int w = tid; w < s.nw; w += kThreads)
            s.each(w, [&](float v, int i) {
              if (i >= s.lo && i < s.hi && f(v, i)) n += by_mass ? (unsigned long long)(rs.weight(v) * kUnit) : 1ull;
            });
          return cluster_sum(n, sh_u, slot);
        };
        int flip = 0;
        // the smallest kept key when 1 or masses are summed in descending key order up to ``target``, of the keys >= floor
        auto select = [&](bool by_mass, unsigned long long target, int from, int upto, unsigned long long floor_key,
                          int slot) {
          float lo = -INFINITY, hi = -INFINITY;  // -smallest and largest logit
          for (int w = tid; w < s.nw; w += kThreads)
            s.each(w, [&](float v, int i) {
              const int bin = bin_of(v);
              if (bin < from || bin > upto || i < s.lo || i >= s.hi) return;
              v = fmaxf(v, -INFINITY);
              lo = fmaxf(lo, -v);
              hi = fmaxf(hi, v);
            });
          lo = -cluster_max(lo, sh_f, &slot_f3[slot][0]);
          hi = cluster_max(hi, sh_f, &slot_f3[slot][1]);
          unsigned long long before = total_of(by_mass, &slot_u[slot * 2 + 1], [&](float v, int i) {
            return v > hi && rank_key(v, i) >= floor_key;
          });
          // bits that differ: of the logits, then of the tokens
          const uint32_t diff = order_key(lo + 0.f) ^ order_key(hi + 0.f);
          const int token_bits = 32 - __clz(V - 1);
          int bits = diff != 0 ? 64 - __clz(diff) : token_bits;
          const unsigned long long top_key = (unsigned long long)order_key(hi + 0.f) << 32 | 0xffffffffull;
          unsigned long long prefix = bits < 64 ? top_key >> bits << bits : 0ull;
          while (bits > 0) {
            const int nb = min(8, bits > 32 ? bits - 32 : bits), shift = bits - nb;
            const unsigned int bin_mask = (1u << nb) - 1;
            unsigned long long* h = hist_m[flip];
            unsigned int* hc = hist_c[flip];
            if (tid < 256) h[tid] = 0, hc[tid] = 0;
            __syncthreads();
            for (int w = tid; w < s.nw; w += kThreads)
              s.each(w, [&](float v, int i) {
                if (!(v <= hi) && !isnan(v)) return;
                if (v < lo || i < s.lo || i >= s.hi) return;
                const unsigned long long key = rank_key(v, i);
                if (key < floor_key || (bits < 64 ? (key ^ prefix) >> bits : 0ull) != 0) return;
                const unsigned int bin = (unsigned int)(key >> shift) & bin_mask;
                atomicAdd(&hc[bin], 1u);
                if (by_mass) atomicAdd(&h[bin], (unsigned long long)(rs.weight(v) * kUnit));
              });
            __syncthreads();
            if (CL > 1) nvb::cluster_sync();
            // every CTA adds up the cluster's bins and finds the same one
            if (tid < 256) {
              unsigned long long v = 0;
              unsigned int c = 0;
              for (uint32_t i = 0; i < CL; ++i) {
                c += CL > 1 ? peer_load(&hc[tid], i) : hc[tid];
                if (by_mass) v += CL > 1 ? peer_load(&h[tid], i) : h[tid];
              }
              keys[tid] = by_mass ? v : c;
              keys[256 + tid] = c;
            }
            __syncthreads();
            if (warp == 0) {  // lane: 8 bins from the top
              unsigned long long own = 0;
#pragma unroll
              for (int i = 0; i < 8; ++i) own += keys[255 - lane * 8 - i];
              unsigned long long incl = own;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
              }
              const unsigned hit = __ballot_sync(0xffffffffu, before + incl >= target);
              if (lane == (hit != 0 ? __ffs(hit) - 1 : 31)) {
                unsigned long long cum = before + incl - own;
                int bin = 255 - lane * 8;
                for (; bin > 248 - lane * 8 && cum + keys[bin] < target; --bin) cum += keys[bin];
                sel_u[0] = prefix & ~(((unsigned long long)bin_mask) << shift) | ((unsigned long long)bin << shift);
                sel_u[1] = cum;
                sel[1] = keys[256 + bin] <= 1;
              }
            }
            __syncthreads();
            prefix = sel_u[0] >> shift << shift;
            before = sel_u[1];
            const bool alone = sel[1] != 0;
            bits = shift;
            if (bits == 32 && token_bits < 32) {  // token bits above the vocabulary's are ones
              bits = token_bits;
              prefix |= 0xffffffffull >> token_bits << token_bits;
            }
            flip ^= 1;  // the peers may still read the other one
            __syncthreads();
            if (alone) break;  // no other key begins like this
          }
          return prefix;
        };
        const int sure_k = sel[0], sure_p = sel[1], may_p = sel[2];
        __syncthreads();
        if (cut_k) cut = select(false, (unsigned long long)k, max(0, sure_k - 1), min(kBins - 1, sure_k + 1), 0, 0);
        if (cut_p) {
          const unsigned long long total =
              total_of(true, &slot_u[0], [&](float v, int i) { return rank_key(v, i) >= cut; });
          const double want = (double)total * (double)top;
          const unsigned long long target = want > 1.0 ? (unsigned long long)ceil(want) : 1ull;  // the first always stays
          cut = max(cut, select(true, target, cut_k ? 0 : max(0, may_p - 1), cut_k ? kBins - 1 : min(kBins - 1, sure_p + 1),
                                cut, 1));
        }
        double z = 0.0;
        for (int w = tid; w < s.nw; w += kThreads) {
          float part = 0.f;
          s.each(w, [&](float v, int i) {
            if (rank_key(v, i) >= cut) part += rs.weight(v);
          });
          z += part;
        }
        Z = cluster_sum(z, sh_d, &slot_d[1]);
      }
    }
  }
  if (rank == 0 && tid == 0) {
    a.cut[r] = cut;
    a.row_max[r] = m;
  }
  if (r + 1 < rows.y) {  // the draft
    bool near = false;
    double w = 0.0, uq = 0.0;
    if (rank == 0) {
      const int dr = a.probs != nullptr ? draft_row(a, b, r, sh_i) : 0;
      const long d = a.ids[r + 1];
      if (a.probs != nullptr && dr >= a.D) {
        if (tid == 0) nvb::record_error(a.err, nvb::kErrBadArgument);
      } else if (d >= 0 && d < V) {
        const float v = to_float(x[d]);
        if (rank_key(v, (int)d) >= cut) w = rs.weight64(v, table);
        uq = a.uniform(r) * (a.probs != nullptr ? (double)a.probs[dr * a.probs_ld + d] : 1.0);
      }
      near = fabs(uq * Z - w) <= 1e-4 * w;  // too near for a sum of 32-bit weights
      if (tid == 0) sel[0] = near;
    }
    if (CL > 1) {
      nvb::cluster_sync();
      near = peer_load(&sel[0], 0) != 0;
      if (near) cut = rank == 0 ? cut : 0;  // only rank 0 needs to know the cut from here
    }
    if (near) {
      if (CL > 1) {
        if (rank == 0 && tid == 0) sel_u[0] = cut;
        nvb::cluster_sync();
        cut = peer_load(&sel_u[0], 0);
      }
      double z64 = 0.0;
      for (int q = tid; q < s.nw; q += kThreads)
        s.each(q, [&](float v, int i) {
          if (rank_key(v, i) >= cut && i >= s.lo && i < s.hi) z64 += rs.weight64(v, table);
        });
      Z = cluster_sum(z64, sh_d, &slot_d[2]);
    }
    if (rank == 0 && tid == 0) a.accept[r] = uq * Z < w;
  }
  if (CL > 1) nvb::cluster_sync();  // nobody leaves while its shared memory may be read
}

// One cluster per sequence: the accepted drafts and the drawn token.  Weights and sums in 64 bits: the token depends on
// which side of a sum the uniform falls, and a row has as many sums as tokens.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_draw_kernel(const VerifyArgs a) {
  nvb::pdl_wait();
  nvb::pdl_trigger();
  extern __shared__ __align__(128) uint8_t buf[];
  __shared__ uint64_t bar;
  __shared__ double sh_d[32], slot_d, table[kTable], warp_sum_sh[2][kWarps], all_sh[kMaxCluster * kWarps + 1];
  __shared__ int sh_i[32];
  const int b = blockIdx.x / cluster_size(), tid = threadIdx.x, V = a.V, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = nvb::cluster_ctarank(), CL = cluster_size();
  const int2 rows = seq_rows(a, b);
  const int n = rows.y - rows.x;
  int64_t* out = a.tokens + (long)b * a.max_q;
  if (n <= 0) {  // the whole cluster
    if (rank == 0) {
      for (int j = tid; j < a.max_q; j += kThreads) out[j] = -1;
      if (tid == 0) {
        a.counts[b] = 0;
        if (n < 0) nvb::record_error(a.err, nvb::kErrBadArgument);
      }
    }
    return;
  }
  int acc = n - 1;  // accepted drafts: up to the first refusal
  for (int j0 = 0; j0 < n - 1; j0 += 32) {
    const bool no = j0 + lane < n - 1 && !a.accept[rows.x + j0 + lane];
    const unsigned refused = __ballot_sync(0xffffffffu, no);
    if (refused != 0) {
      acc = j0 + __ffs(refused) - 1;
      break;
    }
  }
  const int r = rows.x + acc;
  const bool rejected = acc < n - 1;
  const Slice<T> s = load_slice(reinterpret_cast<const T*>(a.logits) + r * a.ld, V, buf, &bar);
  const unsigned long long cut = a.cut[r];
  const RowScale rs(a.row_max[r], a.softcap, a.temps[b]);
  const int dr = rejected && a.probs != nullptr ? draft_row(a, b, r, sh_i) : 0;
  const float* q = rejected && a.probs != nullptr && dr < a.D ? a.probs + dr * a.probs_ld : nullptr;
  const long drafted = rejected && a.probs == nullptr ? a.ids[r + 1] : -1;
  fill_table(table);
  finish_slice(s, &bar, a.err);
  const bool simple = cut == 0 && rs.simple();
  const float cut_logit = cut == 0 ? -INFINITY : key_logit(cut);
  constexpr int PER = Slice<T>::PER;
  // weights of a word's tokens (what a slice's first and last word hold besides weighs nothing)
  auto word_weights = [&](int w, double (&l)[PER]) {
    const uint4 raw = reinterpret_cast<const uint4*>(s.words)[w];
    const T* e = reinterpret_cast<const T*>(&raw);
    if (simple) {
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = rs.weight64_simple(to_float(e[j]), table);
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float v = to_float(e[j]);  // with a cut most tokens are below its logit
        l[j] = v >= cut_logit && rank_key(v, s.first + w * PER + j) >= cut ? rs.weight64(v, table) : 0.0;
      }
    }
  };
  double Zinv = 1.0;
  if (q != nullptr) {  // p - q needs p itself
    double z = 0.0, l[PER];
    for (int w = tid; w < s.nw; w += kThreads) {
      word_weights(w, l);
#pragma unroll
      for (int j = 0; j < PER; ++j) z += l[j];
    }
    const double Z = cluster_sum(z, sh_d, &slot_d);
    Zinv = Z > 0.0 ? 1.0 / Z : 0.0;
  }
  const bool q_aligned = q != nullptr && ((reinterpret_cast<uintptr_t>(q) + 4 * (long)s.first) & 15) == 0;
  // what is left of a word's tokens to draw from; plain: the probabilities themselves
  auto word_left = [&](int w, bool plain, double (&l)[PER]) {
    word_weights(w, l);
    if (plain) return;
    const int i0 = s.first + w * PER;
    if (q == nullptr) {
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = i0 + j == drafted ? 0.0 : l[j];
    } else {
      float qv[PER];
      if (q_aligned && i0 >= s.lo && i0 + PER <= s.hi) {
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(q + i0 + j);
          qv[j] = v.x, qv[j + 1] = v.y, qv[j + 2] = v.z, qv[j + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) qv[j] = i0 + j >= s.lo && i0 + j < s.hi ? q[i0 + j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = l[j] > 0.0 ? fmax(0.0, l[j] * Zinv - (double)qv[j]) : 0.0;
    }
  };
  // warps own consecutive words, lanes one word at a time
  const int per = (s.nw + kWarps - 1) / kWarps, w0 = min(s.nw, warp * per), w1 = min(s.nw, w0 + per);
  for (int plain = rejected ? 0 : 1; plain < 2; ++plain) {
    // plain: the probabilities themselves, also when nothing is left of p - q
    double sum = 0.0, l[PER];
    for (int w = w0 + lane; w < w1; w += 32) {
      word_left(w, plain != 0, l);
#pragma unroll
      for (int j = 0; j < PER; ++j) sum += l[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) warp_sum_sh[plain][warp] = sum;
    __syncthreads();
    if (CL > 1) nvb::cluster_sync();
    // sums before each warp of the cluster, in token order; every CTA computes the same ones
    const int nws = (int)CL * kWarps;
    if (tid < nws) all_sh[tid] = CL > 1 ? peer_load(&warp_sum_sh[plain][tid % kWarps], tid / kWarps) : warp_sum_sh[plain][tid];
    __syncthreads();
    if (tid == 0) {
      double c = 0.0;  // one after the other: the sums never decrease
      for (int i = 0; i < nws; i += kWarps) {
        double v[kWarps];
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v[k] = all_sh[i + k];
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          all_sh[i + k] = c;
          c += v[k];
        }
      }
      all_sh[nws] = c;
    }
    __syncthreads();
    const double total = all_sh[nws];
    if (total > 0.0) {
      // below total whatever the uniform is, so some token exceeds it
      const double want = fmin(fmax(a.uniform(rows.y - 1), 0.0), 1.0 - 2.220446049250313e-16) * total;
      const int me = (int)rank * kWarps + warp;
      double c = all_sh[me];
      if (c <= want && all_sh[me + 1] > want) {  // this warp's words hold it
        int tok = -1;
        for (int wb = w0; wb < w1; wb += 32) {
          double mine = 0.0;
          if (wb + lane < w1) {
            word_left(wb + lane, plain != 0, l);
#pragma unroll
            for (int j = 0; j < PER; ++j) mine += l[j];
          }
          double incl = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
          }
          const unsigned over = __ballot_sync(0xffffffffu, mine > 0.0 && c + incl > want);
          const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0);
          const int src = over != 0 ? __ffs(over) - 1 : some != 0 ? 31 - __clz(some) : -1;
          int cand = -1;
          if (lane == src) {
            double d = c + incl - mine;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              if (l[j] > 0.0 && !(cand >= 0 && d > want)) cand = s.first + (wb + lane) * PER + j;
              d += l[j];
            }
          }
          if (src >= 0) tok = __shfl_sync(0xffffffffu, cand, src);
          if (over != 0) break;
          c += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) out[acc] = tok < 0 ? 0 : tok;
      }
      break;
    }
    if (plain == 1 && rank == 0 && tid == 0) out[acc] = 0;  // no logit above -inf
  }
  if (rank == 0) {
    for (int j = tid; j < a.max_q; j += kThreads)
      if (j != acc) out[j] = j < acc ? a.ids[rows.x + j + 1] : -1;
    if (tid == 0) a.counts[b] = acc + 1;
  }
  if (CL > 1) nvb::cluster_sync();  // nobody leaves while its shared memory may be read
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
  TORCH_CHECK(V >= 1 && V <= kMaxVocab, "the vocabulary must have 1 to 327680 tokens");
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
  auto scratch = at::empty({R * 2}, ids.options());  // cut, then largest logit and acceptance
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
  a.row_max = reinterpret_cast<float*>(scratch.data_ptr<int64_t>() + R);
  a.accept = reinterpret_cast<int*>(a.row_max + R);
  a.err = err.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool wide = logits.scalar_type() == at::kFloat;
  const int64_t width = wide ? 4 : 2;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // CTAs per row: two of them fit an SM (their slices at most 80 KB), more while SMs would idle
  auto cluster_for = [&](int64_t count) {
    int64_t n = 1;
    while (n < kMaxCluster && (V * width > n * 80 * 1024 || count * n * 2 <= sms)) n *= 2;
    return n;
  };
  auto run = [&](auto kern, int64_t count) {
    const int64_t n = cluster_for(count);
    const size_t smem = (size_t)(((V + n - 1) / n + 7) / 8 * 8 * width + 32);
    TORCH_CHECK(smem <= 190 * 1024, "the vocabulary does not fit the shared memory of a cluster");
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    C10_CUDA_CHECK(nvb::launch_cluster(kern, dim3((unsigned)(n * count)), dim3(kThreads), smem, stream, (unsigned)n, a));
  };
  if (R > 0) {
    if (wide) run(verify_rows_kernel<float>, R);
    else run(verify_rows_kernel<bf16>, R);
  }
  if (wide) run(verify_draw_kernel<float>, B);
  else run(verify_draw_kernel<bf16>, B);
  return {tokens, counts, R > 0 ? 2 : 1};
}
