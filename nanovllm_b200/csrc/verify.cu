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
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>
#include <tuple>

#include "common.cuh"
#include "launch.h"

namespace {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr double kLog2e64 = 1.4426950408889634074;
constexpr int kMaxVocab = 327680;  // 32-bit logits of a row in the shared memory of eight CTAs
constexpr int kMaxCluster = 16;
constexpr int kList = 256;     // tokens that a cut is found among by ranking
constexpr int kOwnList = 256;  // of one CTA
constexpr int kTop = 64;     // largest top_k that the list is tried for

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
  // the kept set where it is a list of at most kList tokens: their number (else 0), tokens in order, weights
  int* kept_n;
  int* kept_tok;
  double* kept_w;
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

// 2^(d c) in 64 bits (relative error below 1e-12) for an exponent in [-1000, 0]: it is k / 128 + r, with a table of
// 2^(k / 128) and the exponential series for 2^r, |r| <= R = 1/256, whose fourth term a r^4 is taken as a (R^2 r^2 - R^4 / 8)
// (off by at most a R^4 / 8 = 2.8e-13).
constexpr int kTable = 128;
template <bool IN_RANGE = false>  // true: the exponent is known to lie above -1000
NV_DEVICE double exp2_64(double d, double c, const double* table) {
  const double magic = 52776558133248.0;  // 1.5 * 2^45: the last bit of a sum with it is 1/128
  const double t = fma(d, c, magic);
  const double r = fma(d, c, magic - t);
  const int k = IN_RANGE ? __double2loint(t) : max(__double2loint(t), -1000 * kTable);
  double p = 5.550410866482158e-2;
  p = fma(p, r, 2.402265069591007e-1 + 9.618129107628477e-3 / 65536);
  p = fma(p, r, 6.931471805599453e-1);
  p = fma(p, r, 1.0 - 9.618129107628477e-3 / 65536 / 65536 / 8) * table[k & (kTable - 1)];
  return __hiloint2double(__double2hiint(p) + (k >> 7) * (1 << 20), __double2loint(p));
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
    return x >= floor64 ? floored64(x, table) : 0.0;  // NaN, -inf: 0
  }
  // the same where x >= floor64; else 2^-996 (the floor lies 690 log2(e) < 996 below the largest)
  NV_DEVICE double floored64(float x, const double* table) const {
    return exp2_64<true>((double)fmaxf(x, floor64) - m64, c64, table);
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

NV_DEVICE uint4 peer_load4(const uint32_t* p, uint32_t rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(nvb::map_peer(nvb::smem_u32(p), rank))
               : "memory");
  return v;
}

template <typename T>
NV_DEVICE void peer_store(T* p, uint32_t rank, T v) {
  const uint32_t at = nvb::map_peer(nvb::smem_u32(p), rank);
  if constexpr (sizeof(T) == 8)
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(*reinterpret_cast<unsigned long long*>(&v)) : "memory");
  else
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(*reinterpret_cast<uint32_t*>(&v)) : "memory");
}

// Reductions over the cluster with one barrier of it: the CTAs' totals go into every CTA's table, each thread then reads
// its own CTA's, in the same order everywhere.  Two tables in turn: whoever writes one again has passed a barrier that
// everybody reached after reading it.
constexpr int kValues = 6;
struct Tables {
  double v[2][kValues][kMaxCluster], warps[kValues][kWarps];
};
template <int N, bool MAX, typename T>
NV_DEVICE void cluster_reduce(T (&v)[N], Tables& tables, int& turn) {
  static_assert(N <= kValues && N * kMaxCluster <= kThreads);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = (int)cluster_size(), rank = (int)nvb::cluster_ctarank();
  T* t = reinterpret_cast<T*>(tables.v[turn & 1]);
  T* sh = reinterpret_cast<T*>(tables.warps);
  ++turn;
  auto join = [](T a, T b) { return MAX ? (a > b ? a : b) : a + b; };
#pragma unroll
  for (int k = 0; k < N; ++k) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] = join(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
    if (lane == 0) sh[k * kWarps + warp] = v[k];
  }
  __syncthreads();
  if (tid < N * n) {
    const int k = tid / n, peer = tid % n;
    T x = sh[k * kWarps];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) x = join(x, sh[k * kWarps + w]);
    peer_store(&t[k * kMaxCluster + rank], peer, x);
  }
  nvb::cluster_sync();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    T x = t[k * kMaxCluster + (lane < n ? lane : 0)];
    if (lane >= n && !MAX) x = (T)0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = join(x, __shfl_xor_sync(0xffffffffu, x, o));
    v[k] = x;
  }
}

// The cluster's CTAs are there once each has arrived: waited for before the first access to another's shared memory.
NV_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
NV_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

NV_DEVICE int block_sum(int v, int* sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  int r = 0;
  for (int i = 0; i < kWarps; ++i) r += sh[i];
  return r;
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

// The largest logit of this thread's words (NaN is passed over).
template <typename T>
NV_DEVICE float slice_max(const Slice<T>& s) {
  float m = -INFINITY;
  if constexpr (sizeof(T) == 2) {  // two at a time
    __nv_bfloat162 acc = __float2bfloat162_rn(-INFINITY);
    for (int w = threadIdx.x; w < s.nw; w += kThreads) {
      const uint4 v = reinterpret_cast<const uint4*>(s.words)[w];
      const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&v);
      acc = __hmax2(acc, __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3])));
    }
    m = fmaxf(m, fmaxf(__low2float(acc), __high2float(acc)));
  } else {
    for (int w = threadIdx.x; w < s.nw; w += kThreads) s.each(w, [&](float v, int) { m = fmaxf(m, v); });
  }
  return m;
}

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
// shared memory, every pass after the load reads it there.
//   no cut     each CTA's maximum and sum of weights against it, joined in rank 0 by one exchange
//   top_k 1    the lowest token of the largest logit, by one exchange
//   cuts       some hundred of the largest logits are ranked and walked, in one CTA; a cut that lies beyond them (a flat
//              row, a large top_k) is found by a histogram, where that does not reach it by passes that sum what lies
//              above three thresholds each
// Few rows are bound by the chain of these steps (5 rows of 151936 tokens with a top_p: 14 us, of which 3 us each are the
// load, the pass that sums and lists, and the ranking), many by the issue of instructions (577 rows without a cut: 60 us,
// 2.9 TB/s of logits, 13 instructions a token with the exponential's).
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) verify_rows_kernel(const VerifyArgs a) {
  nvb::pdl_wait();
  nvb::pdl_trigger();
  extern __shared__ __align__(128) uint8_t buf[];
  __shared__ uint64_t bar;
  __shared__ Tables red;
  __shared__ double table[kTable], sh_d[kWarps];
  __shared__ float sh_f[kWarps], threshold_sh;
  __shared__ int sh_i[kWarps];
  __shared__ unsigned int n_list, n_gather, eq_sh[2][kMaxCluster * kWarps];
  __shared__ unsigned long long keys[kOwnList], found_sh[2];
  // the threads' maxima, then rank 0's list (keys, and weights in order), then a histogram
  __shared__ __align__(16) double pool[2 * kList];
  __shared__ double hit_mass;
  __shared__ int hit_bin, hit_count;
  __shared__ unsigned int told, tie;  // tie: 1 when top_p falls on a sum of the list, 2 once that is resolved
  float* maxima = reinterpret_cast<float*>(pool);
  const int r = blockIdx.x / cluster_size(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.V;
  const uint32_t rank = nvb::cluster_ctarank(), CL = cluster_size();
  cluster_arrive();
  int turn = 0;
  auto sum1 = [&](double v) {
    double x[1] = {v};
    cluster_reduce<1, false>(x, red, turn);
    return x[0];
  };
  const T* x = reinterpret_cast<const T*>(a.logits) + r * a.ld;
  const Slice<T> s = load_slice(x, V, buf, &bar);
  const int b = seq_of_row(a.cu_q, a.B, r);
  const int2 rows = seq_rows(a, b);
  const bool in_seq = r >= rows.x && r < rows.y;
  const int k = a.topk[b];
  const float top = a.topp[b], temp = a.temps[b];
  // the draft's logit, probability and uniform come while the row does
  const bool drafted = in_seq && r + 1 < rows.y;
  long d = -1;
  float d_logit = 0.f;
  double uq = 0.0;
  if (drafted && rank == 0) {
    const int dr = a.probs != nullptr ? draft_row(a, b, r, sh_i) : 0;
    d = a.ids[r + 1];
    if (a.probs != nullptr && (dr < 0 || dr >= a.D)) {
      if (tid == 0) nvb::record_error(a.err, nvb::kErrBadArgument);
      d = -1;
    }
    if (d >= V) d = -1;
    if (d >= 0) {
      d_logit = to_float(x[d]);
      uq = a.uniform(r) * (a.probs != nullptr ? (double)a.probs[dr * a.probs_ld + d] : 1.0);
    }
  }
  fill_table(table);
  if (tid == 0) {
    n_list = n_gather = tie = 0;
    found_sh[0] = found_sh[1] = 0;
  }
  finish_slice(s, &bar, a.err);
  cluster_wait();
  if (!in_seq) return;  // the whole cluster
  const float mine_max = slice_max(s);
  const bool cut_k = k > 0 && k < V, cut_p = top < 1.f;
  unsigned long long cut = 0;
  double Z = 0.0;
  int kept_n = 0;  // rank 0: tokens listed for the draw
  float m;
  if (!cut_k && !cut_p && k != 1 && a.softcap <= 0.f) {
    // ---------------------------------------------------------------- no cut: sums against the CTA's own maximum
    const float mw = nvb::warp_max(mine_max);
    if (lane == 0) sh_f[warp] = mw;
    __syncthreads();
    float mc = sh_f[0];
    for (int i = 1; i < kWarps; ++i) mc = fmaxf(mc, sh_f[i]);
    const RowScale own(mc, 0.f, temp);
    float z4[4] = {0.f, 0.f, 0.f, 0.f};
    const float off = -mc * own.c_hi;
    if (own.simple() && fabsf(off) < 64.f) {  // one product: weights within 1e-5, where near ties are found within 1e-4
      for (int w = tid; w < s.nw; w += kThreads) {
        int j = 0;
        s.each(w, [&](float v, int) { z4[j++ & 3] += exp2f(fmaxf(fmaf(v, own.c_hi, off), -1e30f)); });
      }
    } else if (own.simple()) {
      for (int w = tid; w < s.nw; w += kThreads) {
        int j = 0;
        s.each(w, [&](float v, int) { z4[j++ & 3] += exp2f(own.log_weight_simple(v)); });
      }
    } else if (mc == INFINITY) {
      for (int w = tid; w < s.nw; w += kThreads) s.each(w, [&](float v, int) { z4[0] += v == INFINITY ? 1.f : 0.f; });
    }
    // the CTAs' sums and maxima to rank 0, which alone goes on
    double z = (double)(z4[0] + z4[1]) + (double)(z4[2] + z4[3]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (lane == 0) sh_d[warp] = z;
    __syncthreads();
    if (tid == 0) {
      z = 0.0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) z += sh_d[i];
      peer_store(&red.v[0][0][rank], 0u, z);
      peer_store(&red.v[0][1][rank], 0u, (double)mc);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank != 0) return;  // (nobody writes to another CTA than rank 0)
    cluster_wait();
    const float ml = lane < (int)CL ? (float)red.v[0][1][lane] : -INFINITY;
    const double zl = lane < (int)CL ? red.v[0][0][lane] : 0.0;
    m = nvb::warp_max(ml);
    const RowScale all(m, 0.f, temp);
    Z = zl > 0.0 ? zl * all.weight64(ml, table) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) Z += __shfl_xor_sync(0xffffffffu, Z, o);
  } else if (k == 1) {
    // ---------------------------------------------------------------- greedy: the lowest token among the largest logits
    unsigned long long best[1] = {0};  // of each thread's own largest logit
    for (int w = tid; w < s.nw; w += kThreads) {
      unsigned same = 0;
      int j = 0;
      s.each(w, [&](float v, int) { same |= (v == mine_max ? 1u : 0u) << j++; });
      for (; same != 0; same &= same - 1) {
        const int i = s.first + w * Slice<T>::PER + __ffs(same) - 1;
        if (i >= s.lo && i < s.hi) best[0] = max(best[0], rank_key(mine_max, i));
      }
    }
    cluster_reduce<1, true>(best, red, turn);
    m = best[0] != 0 ? key_logit(best[0]) : -INFINITY;
    cut = m == -INFINITY ? 0 : best[0];
    Z = 1.0;
    kept_n = cut != 0;
    if (rank == 0 && tid == 0 && kept_n != 0) {
      a.kept_tok[(long)r * kList] = (int)(0xffffffffu - (uint32_t)cut);
      a.kept_w[(long)r * kList] = 1.0;
    }
  } else {
    float mv[1] = {mine_max};
    cluster_reduce<1, true>(mv, red, turn);
    m = mv[0];
  }
  const RowScale rs(m, a.softcap, temp);
  const bool simple = rs.simple();
  if (k != 1 && (cut_k || cut_p || a.softcap > 0.f)) {
    const bool cuts = (cut_k || cut_p) && m != -INFINITY;
    // With a cut: this CTA's tokens at or above its threshold, the want_top-th largest of its threads' maxima, so at least
    // that many; the row's list holds every token at or above the largest threshold of the cluster.  That is enough for a
    // top_k when it holds top_k tokens (two times as many are aimed at), for a top_p when it holds the mass.
    const int want_top = min(128, (cut_k ? 2 * min(k, kTop) : 96) / (int)CL + 8);
    if (cuts) {
      maxima[tid] = mine_max;
      __syncthreads();
      if (warp == 0) {
        uint32_t own[kThreads / 32], lo = 0xffffffffu, hi = 0;
#pragma unroll
        for (int j = 0; j < kThreads / 32; ++j) {
          own[j] = order_key(maxima[j * 32 + lane] + 0.f);
          lo = min(lo, own[j]);
          hi = max(hi, own[j]);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        int n_lo = kThreads;
        while (lo < hi && n_lo > want_top + want_top / 4) {  // at least want_top threads at lo, a quarter more will do
          const uint32_t mid = lo + (hi - lo) / 2 + 1;
          int n = 0;
#pragma unroll
          for (int j = 0; j < kThreads / 32; ++j) n += own[j] >= mid;
          n = __reduce_add_sync(0xffffffffu, n);
          if (n >= want_top) lo = mid, n_lo = n;
          else hi = mid - 1;
        }
        if (lane == 0) threshold_sh = key_logit((unsigned long long)lo << 32);
      }
    }
    float threshold = INFINITY;
    if (cuts) {
      __syncthreads();
      threshold = fmaxf(threshold_sh, -FLT_MAX);
    }
    float z4[4] = {0.f, 0.f, 0.f, 0.f};
    // sums the weights and lists what reaches the threshold
    auto pass = [&](auto weight_of) {
      for (int w = tid; w < s.nw; w += kThreads) {
        unsigned listed = 0;
        int j = 0;
        s.each(w, [&](float v, int) {
          z4[j & 3] += weight_of(v);
          listed |= (v >= threshold ? 1u : 0u) << j;
          ++j;
        });
        if (cuts)
          for (; listed != 0; listed &= listed - 1) {
            const int i = w * Slice<T>::PER + __ffs(listed) - 1;
            const unsigned int at = atomicAdd(&n_list, 1u);
            if (at < (unsigned int)kOwnList) keys[at] = rank_key(to_float(s.words[i]), s.first + i);
          }
      }
    };
    if (cuts && cut_k) pass([](float) { return 0.f; });  // the mass of all tokens is not asked for
    else if (simple) pass([&](float v) { return exp2f(rs.log_weight_simple(v)); });
    else pass([&](float v) { return rs.weight(v); });
    Z = sum1((double)(z4[0] + z4[1]) + (double)(z4[2] + z4[3]));
    if (cuts) {
      // (the sum was a barrier of the cluster)
      constexpr double kAll = 4.0 * kMaxVocab;  // more than any count or mass
      // Rank 0: the CTAs' lists as far as they hold logits in [from, to) (to NaN: no end) and keys >= floor, ranked and
      // walked, behind ``count`` tokens of the mass ``mass``.  Kept are the first ``limit`` tokens, while the mass before
      // is below ``want`` (negative: below that share of the mass that the limit leaves).  False when the list is too long
      // or, unless it is ``certain`` to hold the cut, ends before it.
      bool done = false;
      auto walk = [&](float from, float to, unsigned long long floor_key, double count, double mass, double limit,
                      double want, bool certain) {
        unsigned long long* list = reinterpret_cast<unsigned long long*>(pool);
        double* sorted = pool + kList;
        const unsigned int own_n = (uint32_t)lane < CL ? peer_load(&n_list, lane) : 0u;
        if (__any_sync(0xffffffffu, own_n > (unsigned int)kOwnList)) return false;
        for (uint32_t q = warp; q < CL; q += kWarps) {
          const unsigned int nq = __shfl_sync(0xffffffffu, own_n, q);
          for (unsigned int i = lane; i < nq; i += 32) {
            const unsigned long long key = peer_load(&keys[i], q);
            const float v = key_logit(key);
            if (v >= from && !(v >= to) && key >= floor_key) {
              const unsigned int at = atomicAdd(&n_gather, 1u);
              if (at < (unsigned int)kList) list[at] = key;
            }
          }
        }
        __syncthreads();
        const int n = (int)n_gather;
        if (n > kList) return false;
        if (tid == 0 && (n & 1) != 0) list[n] = 0;  // (two keys are read at a time)
        __syncthreads();
        // a token's place is the number of larger keys
        static_assert(kList == kThreads);
        const unsigned long long key = tid < n ? list[tid] : 0;
        int place = 0;
        if (tid < n)
#pragma unroll 4
          for (int j = 0; j < (n + 1) / 2; ++j) {
            const ulonglong2 two = reinterpret_cast<const ulonglong2*>(list)[j];
            place += (two.x > key) + (two.y > key);
          }
        __syncthreads();
        if (tid < n) {
          list[place] = key;
          sorted[place] = count + place < limit ? rs.weight64(key_logit(key), table) : 0.0;
        }
        __syncthreads();
        const double w = tid < n ? sorted[tid] : 0.0;
        double incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        if (lane == 31) sh_d[warp] = incl;
        __syncthreads();
        double base = mass, all = mass;
        for (int i = 0; i < kWarps; ++i) {
          if (i < warp) base += sh_d[i];
          all += sh_d[i];
        }
        const bool enough = certain || (limit < kAll ? count + n >= limit : all >= want);
        if (want < 0.0) want = -want * all;
        else if (!certain && tid < n && fabs(base + incl - w - want) <= 4e-6 * want && tie == 0)
          tie = 1;  // a share of Z, whose 32-bit terms leave it up to 4e-6 off
        const bool keep = tid < n && count + tid < limit && (base + incl - w < want || count + tid == 0.0);
        const int kept = __popc(__ballot_sync(0xffffffffu, keep));  // the kept ones are the first
        if (lane == 0) sh_i[warp] = kept;
        __syncthreads();
        int last = -1;
        for (int i = 0; i < kWarps; ++i) last += sh_i[i];
        if (tid == last) hit_mass = base + incl;
        __syncthreads();
        if (!enough || last < 0) return false;
        cut = list[last];
        Z = hit_mass;
        if (count == 0.0) {  // nothing is kept but what is listed: the list in token order
          kept_n = last + 1;
          if (tid < kept_n) {
            const uint32_t low = (uint32_t)list[tid];
            int at = 0;
#pragma unroll 4
            for (int j = 0; j < kept_n; ++j) at += (uint32_t)list[j] > low;
            a.kept_tok[(long)r * kList + at] = (int)(0xffffffffu - low);
            a.kept_w[(long)r * kList + at] = w;
          }
        }
        return true;
      };
      threshold = nvb::warp_max((uint32_t)lane < CL ? peer_load(&threshold_sh, lane) : -INFINITY);
#pragma unroll 1
      for (;;) {
        if (rank == 0 && (!cut_k || k <= kTop))  // the lists are complete down to the largest threshold
          done = walk(threshold, NAN, 0, 0.0, 0.0, cut_k ? (double)k : kAll,
                      !cut_p ? kAll : cut_k ? -(double)top : (double)top * Z, false);
        if (rank == 0 && tid < (int)CL) peer_store(&told, tid, tie == 1 ? 2u : done ? 1u : 0u);
        nvb::cluster_sync();
        if (told != 2) break;
        // the mass before a token is within that of top Z: once more with Z from 64-bit weights
        double z = 0.0;
#pragma unroll 1
        for (int i = tid; i < s.nw * Slice<T>::PER; i += kThreads) z += rs.weight64(to_float(s.words[i]), table);
        if (tid == 0) n_gather = 0, tie = 2;
        Z = sum1(z);
      }
      if (told == 0) {
        // ------------------------------------------------------------ beyond the list
        // The smallest kept key when 1 or weights are summed in descending order up to ``target``, of the keys >= floor;
        // leaves the kept mass in Z when weights are summed.  A histogram over the first 16 bits of the logits gives the
        // cut's logit (bf16) or a guess of it; from there, or where its bins end above the cut, the range of logits that
        // holds the cut is quartered until few tokens are left in it, or one logit.
        auto select = [&](bool by_mass, double target, float lo, unsigned long long floor_key, int slot) {
          float hi = INFINITY;  // the cut's logit is in [lo, hi), while not ``open`` in [lo, m]
          bool open = false;
          double over[2] = {0.0, 0.0};  // sum and count from hi on
          double in_lo = kAll;          // count from lo on
          float one_logit = NAN, guess_lo = NAN, guess_hi = NAN;
          kept_n = 0;
          {
            uint32_t* bins = reinterpret_cast<uint32_t*>(pool);
            constexpr int kBins = 4 * kThreads;
            static_assert(sizeof(pool) == kBins * 4);
            const uint32_t top_key = order_key(m + 0.f) >> 16;
            reinterpret_cast<uint4*>(bins)[tid] = make_uint4(0, 0, 0, 0);
            if (tid == 0) hit_bin = -1;
            __syncthreads();
            for (int w = tid; w < s.nw; w += kThreads)
              s.each(w, [&](float v, int) {
                const uint32_t at = top_key - (order_key(v + 0.f) >> 16);
                if (v >= lo && at < (uint32_t)kBins) atomicAdd(&bins[at], 1u);
              });
            nvb::cluster_sync();
            uint4 n4 = make_uint4(0, 0, 0, 0);  // every CTA joins all bins, four a thread
            for (uint32_t q = 0; q < CL; q += 4) {
              uint4 v[4];
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i)
                v[i] = q + i < CL ? peer_load4(&bins[4 * tid], q + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) n4.x += v[i].x, n4.y += v[i].y, n4.z += v[i].z, n4.w += v[i].w;
            }
            const uint32_t n[4] = {n4.x, n4.y, n4.z, n4.w};
            // a bin's one value (bf16), or the middle of it
            auto bin_logit = [&](int j) {
              const uint32_t key = top_key - (4 * tid + j);
              const uint32_t low = sizeof(T) == 4 ? 0x7fffu : key >= 0x8000u ? 0u : 0xffffu;
              return key_logit((unsigned long long)(key << 16 | low) << 32);
            };
            double mass[4], sum = 0.0;
            int count = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mass[j] = n[j] == 0 ? 0.0 : by_mass ? n[j] * rs.weight64(bin_logit(j), table) : (double)n[j];
              sum += mass[j];
              count += (int)n[j];
            }
            double incl = sum;
            int incl_n = count;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const double v = __shfl_up_sync(0xffffffffu, incl, o);
              const int c = __shfl_up_sync(0xffffffffu, incl_n, o);
              if (lane >= o) incl += v, incl_n += c;
            }
            if (lane == 31) sh_d[warp] = incl, sh_i[warp] = incl_n;
            __syncthreads();
            int first = 0;  // the first warp that reaches the target, and what lies before it
            double before = 0.0;
            int before_n = 0;
            while (first < kWarps && before + sh_d[first] < target) before += sh_d[first], before_n += sh_i[first], ++first;
            if (warp == first) {
              const unsigned over_t = __ballot_sync(0xffffffffu, before + incl >= target);
              if (lane == __ffs(over_t) - 1) {
                double c = before + (incl - sum);
                int nc = before_n + incl_n - count, j = 0;
                while (j < 3 && c + mass[j] < target) c += mass[j], nc += (int)n[j], ++j;
                hit_bin = 4 * tid + j;
                hit_mass = c;
                hit_count = nc;
              }
            }
            __syncthreads();
            if (hit_bin >= 0) {
              const uint32_t key = top_key - hit_bin;
              if (sizeof(T) == 2) {
                one_logit = key_logit((unsigned long long)(key << 16 | (key >= 0x8000u ? 0u : 0xffffu)) << 32);
                over[0] = by_mass ? hit_mass : (double)hit_count;
                over[1] = (double)hit_count;
              } else {
                auto flush = [](float v) { return fabsf(v) < FLT_MIN ? 0.f : v; };
                guess_lo = fmaxf(lo, flush(key_logit((unsigned long long)(key << 16) << 32)));
                guess_hi = flush(key_logit((unsigned long long)((key + 1) << 16) << 32));
              }
            }
          }
          // sums and counts of the logits at or above each of three
          auto sums = [&](const float (&t)[3], double (&out)[6]) {
            float acc[3] = {0.f, 0.f, 0.f};
            int cnt[3] = {0, 0, 0};
            double all[3] = {0.0, 0.0, 0.0};
            auto pass = [&](auto one_of) {
              for (int w = tid, since = 0; w < s.nw; w += kThreads) {
                s.each(w, [&](float v, int) {
                  const float one = one_of(v);
#pragma unroll
                  for (int q = 0; q < 3; ++q) {
                    acc[q] += v >= t[q] ? one : 0.f;
                    cnt[q] += v >= t[q];
                  }
                });
                if (++since == 4) {  // at most 32 terms in 32 bits
                  since = 0;
#pragma unroll
                  for (int q = 0; q < 3; ++q) all[q] += acc[q], acc[q] = 0.f;
                }
              }
            };
            if (!by_mass) pass([](float) { return 0.f; });
            else if (simple) pass([&](float v) { return exp2f(rs.log_weight_simple(v)); });
            else pass([&](float v) { return rs.weight(v); });
#pragma unroll
            for (int q = 0; q < 3; ++q) {
              out[3 + q] = (double)cnt[q];
              out[q] = by_mass ? all[q] + acc[q] : (double)cnt[q];
            }
            cluster_reduce<6, false>(out, red, turn);
          };
          // the next larger logit (denormals count as zero)
          auto next_up = [](float v) {
            if (fabsf(v) < FLT_MIN) return FLT_MIN;
            const float n = key_logit((unsigned long long)(order_key(v) + 1) << 32);
            return fabsf(n) < FLT_MIN ? 0.f : n;
          };
          const float eps = sizeof(T) == 2 ? 0.00390625f : 1.1920929e-7f;  // half a step, a step of the type
          for (int step = 0; step < 300 && isnan(one_logit); ++step) {
            const bool few = in_lo - over[1] <= (double)kList;
            const float top_v = open ? hi : m;
            const bool narrow = top_v - lo <= eps * fmaxf(fabsf(top_v), fabsf(lo)) || step % 8 == 7;
            if (few || narrow) {  // the smallest and largest logit that are left
              float ends[2] = {-INFINITY, -INFINITY};
              for (int w = tid; w < s.nw; w += kThreads)
                s.each(w, [&](float v, int) {
                  const bool in = v >= lo && (open ? v < hi : v <= m) && v > -INFINITY;
                  ends[0] = fmaxf(ends[0], in ? -v : -INFINITY);
                  ends[1] = fmaxf(ends[1], in ? v : -INFINITY);
                });
              cluster_reduce<2, true>(ends, red, turn);
              if (!(-ends[0] < ends[1])) {
                one_logit = ends[1];
                break;
              }
              if (few) break;
              lo = -ends[0];
              if (ends[1] < INFINITY) hi = next_up(ends[1]), open = true;
            }
            // Three logits between; any of them splits the range.  Equal parts of it, or of the order while it is wide.
            const float up = open ? hi : m, span = 0.25f * up - 0.25f * lo;
            float t[3] = {lo + span, lo + 2.f * span, up - span};
            if (!(up - lo <= 64.f * (1.f + fabsf(m)))) {
              const uint32_t kl = order_key(lo + 0.f), part = (order_key(up + 0.f) - kl) / 4;
#pragma unroll
              for (int q = 0; q < 3; ++q) t[q] = key_logit((unsigned long long)(kl + (q + 1) * part) << 32);
            }
            if (step == 0 && guess_hi > guess_lo) t[0] = guess_lo, t[1] = t[2] = guess_hi;
            else if (!(t[0] > lo)) t[0] = t[1] = t[2] = next_up(lo);
            double f[6];
            sums(t, f);
            if (f[2] >= target) lo = t[2], in_lo = f[5];
            else {
              if (f[1] >= target) lo = t[1], in_lo = f[4], hi = t[2], over[0] = f[2], over[1] = f[5];
              else if (f[0] >= target) lo = t[0], in_lo = f[3], hi = t[1], over[0] = f[1], over[1] = f[4];
              else hi = t[0], over[0] = f[0], over[1] = f[3];
              open = true;
            }
          }
          if (isnan(one_logit)) {  // few tokens: as above
            if (tid == 0) n_list = n_gather = 0;
            __syncthreads();
            for (int w = tid; w < s.nw; w += kThreads)
              s.each(w, [&](float v, int i) {
                if (v >= lo && (!open || v < hi) && v > -INFINITY && i >= s.lo && i < s.hi) {
                  const unsigned int at = atomicAdd(&n_list, 1u);
                  if (at < (unsigned int)kOwnList) keys[at] = rank_key(v, i);
                }
              });
            nvb::cluster_sync();
            if (rank == 0)
              walk(lo, open ? hi : NAN, floor_key, over[1], by_mass ? over[0] : 0.0, by_mass ? kAll : target,
                   by_mass ? target : kAll, true);
            unsigned long long c[1] = {rank == 0 ? cut : 0ull};
            cluster_reduce<1, true>(c, red, turn);
            double z[1] = {rank == 0 && tid == 0 ? Z : 0.0};
            cluster_reduce<1, false>(z, red, turn);
            Z = z[0];
            return c[0];
          }
          // many equal logits: the n_keep lowest tokens among them, by counts of consecutive words, in token order
          const float v_cut = one_logit;
          const double one = by_mass ? rs.weight64(v_cut, table) : 1.0;
          const double missing = ceil((target - over[0]) / fmax(one, 1e-300));
          const int n_keep = (int)fmin(fmax(missing, 1.0), 2.0 * kMaxVocab);
          const int per = (s.nw + kWarps - 1) / kWarps, w0 = min(s.nw, warp * per), w1 = min(s.nw, w0 + per);
          auto equals = [&](int w) {
            int n = 0;
            s.each(w, [&](float v, int i) { n += v == v_cut && i >= s.lo && i < s.hi; });
            return n;
          };
          int n = 0;
          for (int w = w0 + lane; w < w1; w += 32) n += equals(w);
          n = __reduce_add_sync(0xffffffffu, n);
          if ((uint32_t)lane < CL) peer_store(&eq_sh[slot][rank * kWarps + warp], lane, (unsigned int)n);
          nvb::cluster_sync();
          int before = 0;
          for (int i = lane; i < (int)rank * kWarps + warp; i += 32) before += (int)eq_sh[slot][i];
          before = __reduce_add_sync(0xffffffffu, before);
          if (before < n_keep && before + n >= n_keep) {  // the last kept one is in this warp's words
            for (int wb = w0; wb < w1; wb += 32) {
              const int mine = wb + lane < w1 ? equals(wb + lane) : 0;
              int incl = mine;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
              }
              if (before + incl - mine < n_keep && before + incl >= n_keep) {
                int left = n_keep - (before + incl - mine);
                s.each(wb + lane, [&](float v, int i) {
                  if (v == v_cut && i >= s.lo && i < s.hi && --left == 0) found_sh[slot] = rank_key(v, i);
                });
              }
              before += __shfl_sync(0xffffffffu, incl, 31);
            }
          }
          __syncthreads();
          unsigned long long found[1] = {found_sh[slot]};  // when all equal ones stay nobody has it
          cluster_reduce<1, true>(found, red, turn);
          double all_eq = 0.0;
          for (int i = lane; i < (int)CL * kWarps; i += 32) all_eq += (double)eq_sh[slot][i];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) all_eq += __shfl_xor_sync(0xffffffffu, all_eq, o);
          Z = over[0] + one * fmin((double)n_keep, all_eq);
          return found[0] != 0 ? found[0] : (unsigned long long)order_key(v_cut + 0.f) << 32;
        };
        if (cut_k) {
          cut = select(false, (double)k, -FLT_MAX, 0, 0);
          double z = 0.0;
          for (int w = tid; w < s.nw; w += kThreads) {
            float part = 0.f;
            s.each(w, [&](float v, int i) {
              if (rank_key(v, i) >= cut) part += rs.weight(v);
            });
            z += part;
          }
          Z = sum1(z);
        }
        if (cut_p) {
          const unsigned long long floor_key = cut;
          // below the largest by log V + 18 temperatures all tokens together weigh less than 2^-25
          const float lo = simple ? fmaxf(m - temp * (logf((float)V) + 18.f), -FLT_MAX) : -FLT_MAX;
          cut = max(floor_key, select(true, (double)top * Z, cut_k ? key_logit(cut) : lo, floor_key, 1));
        }
      }
    }
  }
  if (rank != 0) return;  // (no CTA touches another's shared memory behind the last barrier)
  if (tid == 0) {
    a.cut[r] = cut;
    a.row_max[r] = m;
    a.kept_n[r] = kept_n;
  }
  if (drafted) {
    const double w = d >= 0 && rank_key(d_logit, (int)d) >= cut ? rs.weight64(d_logit, table) : 0.0;
    if (w > 0.0 && fabs(uq * Z - w) <= 1e-4 * w) {  // too near for a sum of 32-bit weights: the row once more
      double z = 0.0;
      for (int i = tid; i < V; i += kThreads) {
        const float v = to_float(x[i]);
        if (rank_key(v, i) >= cut) z += rs.weight64(v, table);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      __syncthreads();
      if (lane == 0) sh_d[warp] = z;
      __syncthreads();
      Z = 0.0;
      for (int i = 0; i < kWarps; ++i) Z += sh_d[i];
    }
    if (tid == 0) a.accept[r] = uq * Z < w;
  }
}

// One cluster per sequence: the accepted drafts and the drawn token.  Weights and sums in 64 bits: the token depends on
// which side of a sum the uniform falls, and a row has as many sums as tokens.  Where the kept tokens are listed one CTA
// draws from the list (6 us for any batch that fits the GPU at once); else the row is summed, once for p and once more
// for p - q: 128 rows of 151936 tokens with drafters' distributions 70 us, bound by the issue of 28 instructions a token
// and pass.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) verify_draw_kernel(const VerifyArgs a) {
  nvb::pdl_wait();
  nvb::pdl_trigger();
  extern __shared__ __align__(128) uint8_t buf[];
  __shared__ uint64_t bar;
  __shared__ Tables red;
  __shared__ double table[kTable], all_sh[2][kMaxCluster * kWarps + 1], sub_sh[kWarps];
  __shared__ int sh_i[kWarps], first_sh[kWarps], last_sh[kWarps];
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
  auto finish = [&] {
    for (int j = tid; j < a.max_q; j += kThreads)
      if (j != acc) out[j] = j < acc ? a.ids[rows.x + j + 1] : -1;
    if (tid == 0) a.counts[b] = acc + 1;
  };
  const int kept_n = a.kept_n[r];
  if (kept_n > 0) {
    // ---------------------------------------------------------------- the kept tokens are listed: one CTA, a token a thread
    if (rank != 0) return;
    bool here = tid < kept_n;
    const int tok = here ? a.kept_tok[(long)r * kList + tid] : 0;
    here = here && tok >= 0 && tok < V;  // (a row that no sequence of a malformed cu_q holds has no list)
    const double w = here ? a.kept_w[(long)r * kList + tid] : 0.0;
    double l = w;
    // inclusive sums over the CTA; the total in ``total``
    double total = 0.0;
    auto scan = [&](double v) {
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
      }
      __syncthreads();
      if (lane == 31) sub_sh[warp] = v;
      __syncthreads();
      double base = 0.0;
      total = 0.0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < warp) base += sub_sh[i];
        total += sub_sh[i];
      }
      return base + v;
    };
    if (rejected) {
      if (a.probs != nullptr) {
        const int dr = draft_row(a, b, r, sh_i);
        scan(w);
        if (dr >= 0 && dr < a.D && here) l = fmax(0.0, w * (1.0 / total) - (double)a.probs[dr * a.probs_ld + tok]);
      } else if (here && a.ids[r + 1] == tok) {
        l = 0.0;
      }
    }
    double incl = scan(l);
    if (!(total > 0.0)) {  // nothing is left of p - q: the probabilities themselves
      l = w;
      incl = scan(l);
    }
    const double want = fmin(fmax(a.uniform(rows.y - 1), 0.0), 1.0 - 2.220446049250313e-16) * total;
    // the first token whose sum exceeds ``want``; sums that end a rounding before it: the last token with weight
    const unsigned over = __ballot_sync(0xffffffffu, l > 0.0 && incl > want);
    const unsigned some = __ballot_sync(0xffffffffu, l > 0.0);
    if (lane == 0) {
      first_sh[warp] = over != 0 ? warp * 32 + __ffs(over) - 1 : kThreads;
      last_sh[warp] = some != 0 ? warp * 32 + 31 - __clz(some) : 0;
    }
    __syncthreads();
    int pick = kThreads, last = 0;
    for (int i = 0; i < kWarps; ++i) pick = min(pick, first_sh[i]), last = max(last, last_sh[i]);
    if (tid == (pick < kThreads ? pick : last)) out[acc] = tok;
    finish();
    return;
  }
  cluster_arrive();
  const Slice<T> s = load_slice(reinterpret_cast<const T*>(a.logits) + r * a.ld, V, buf, &bar);
  const unsigned long long cut = a.cut[r];
  const RowScale rs(a.row_max[r], a.softcap, a.temps[b]);
  const int dr = rejected && a.probs != nullptr ? draft_row(a, b, r, sh_i) : 0;
  const float* q = rejected && a.probs != nullptr && dr >= 0 && dr < a.D ? a.probs + dr * a.probs_ld : nullptr;
  const long drafted = rejected && a.probs == nullptr ? a.ids[r + 1] : -1;
  if (q != nullptr)  // p is summed before q is read: q comes nearer meanwhile
    for (int i = s.lo + tid * 32; i < s.hi; i += kThreads * 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + i));
  fill_table(table);
  finish_slice(s, &bar, a.err);
  cluster_wait();
  const bool simple = cut == 0 && rs.simple();
  const float cut_logit = cut == 0 ? -INFINITY : key_logit(cut);
  constexpr int PER = Slice<T>::PER;
  const int cut_tok = (int)(0xffffffffu - (uint32_t)cut);
  // which of a word's tokens are kept, one bit each
  auto word_kept = [&](int w) {
    unsigned kept = 0;
    int j = 0;
    s.each(w, [&](float v, int i) {
      kept |= (v >= cut_logit && v > -INFINITY && (v != cut_logit || i <= cut_tok) ? 1u : 0u) << j;
      ++j;
    });
    return kept;
  };
  // weights of a word's tokens (what a slice's first and last word hold besides weighs nothing); false: nothing
  auto word_weights = [&](int w, double (&l)[PER]) {
    const uint4 raw = reinterpret_cast<const uint4*>(s.words)[w];
    const T* e = reinterpret_cast<const T*>(&raw);
    if (simple) {
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = rs.weight64_simple(to_float(e[j]), table);
    } else {
      const unsigned kept = word_kept(w);  // with a cut most words lie below its logit
      if (kept == 0) return false;
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = (kept >> j & 1u) != 0 ? rs.weight64(to_float(e[j]), table) : 0.0;
    }
    return true;
  };
  double Zinv = 1.0;
  if (q != nullptr) {  // p - q needs p itself
    double z = 0.0;
    if (simple) {
      for (int w = tid; w < s.nw; w += kThreads)
        s.each(w, [&](float v, int) {
          const double e = rs.floored64(v, table);
          if (v >= rs.floor64) z += e;
        });
    } else {
      for (int w = tid; w < s.nw; w += kThreads)
        for (unsigned kept = word_kept(w); kept != 0; kept &= kept - 1)
          z += rs.weight64(to_float(s.words[w * PER + __ffs(kept) - 1]), table);
    }
    double zs[1] = {z};
    int turn = 0;
    cluster_reduce<1, false>(zs, red, turn);
    const double Z = zs[0];
    Zinv = Z > 0.0 ? 1.0 / Z : 0.0;
  }
  const bool q_aligned = q != nullptr && ((reinterpret_cast<uintptr_t>(q) + 4 * (long)s.first) & 15) == 0;
  // the draft's probabilities of a word's tokens
  auto word_q = [&](int i0, float (&qv)[PER]) {
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
  };
  // what is left of a word's tokens to draw from; plain: the probabilities themselves
  auto word_left = [&](int w, bool plain, double (&l)[PER]) {
    if (!word_weights(w, l)) return false;
    if (plain) return true;
    const int i0 = s.first + w * PER;
    if (q == nullptr) {
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = i0 + j == drafted ? 0.0 : l[j];
    } else {
      float qv[PER];
      word_q(i0, qv);
#pragma unroll
      for (int j = 0; j < PER; ++j) l[j] = l[j] > 0.0 ? fmax(0.0, fma(l[j], Zinv, -(double)qv[j])) : 0.0;
    }
    return true;
  };
  auto warp_left = [&](int wa, int wz, bool plain) {  // of words [wa, wz)
    double sum = 0.0, l[PER];
    if (simple && (q == nullptr || plain)) {  // the same terms with less to select
      const int skip = plain || drafted < 0 || drafted >= V ? -1 : (int)drafted;
      for (int w = wa + lane; w < wz; w += 32)
        s.each(w, [&](float v, int i) {
          const double e = rs.floored64(v, table);
          if (v >= rs.floor64 && i != skip) sum += e;
        });
    } else if (simple) {
      for (int w = wa + lane; w < wz; w += 32) {
        float qv[PER];
        word_q(s.first + w * PER, qv);
        int j = 0;
        s.each(w, [&](float v, int) {
          const double left = fma(rs.floored64(v, table), Zinv, -(double)qv[j++]);
          if (left > 0.0 && v >= rs.floor64) sum += left;
        });
      }
    } else if (cut != 0) {  // a lane takes its kept tokens one by one: they are few
      for (int w = wa + lane; w < wz; w += 32)
        for (unsigned kept = word_kept(w); kept != 0; kept &= kept - 1) {
          const int at = w * PER + __ffs(kept) - 1, i = s.first + at;
          const double e = rs.weight64(to_float(s.words[at]), table);
          if (plain) sum += e;
          else if (q == nullptr) sum += i == drafted ? 0.0 : e;
          else sum += fmax(0.0, fma(e, Zinv, -(double)q[i]));
        }
    } else {
      for (int w = wa + lane; w < wz; w += 32)
        if (word_left(w, plain, l))
#pragma unroll
          for (int j = 0; j < PER; ++j) sum += l[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
  };
  // warps own consecutive words, lanes one word at a time
  const int per = (s.nw + kWarps - 1) / kWarps, w0 = min(s.nw, warp * per), w1 = min(s.nw, w0 + per);
  for (int plain = rejected ? 0 : 1; plain < 2; ++plain) {
    // plain: the probabilities themselves, also when nothing is left of p - q
    const double sum = warp_left(w0, w1, plain != 0);
    // every warp's sum to every CTA: the sums before each warp of the cluster, in token order, the same everywhere
    if ((uint32_t)lane < CL) peer_store(&all_sh[plain][rank * kWarps + warp], lane, sum);
    nvb::cluster_sync();
    const int nws = (int)CL * kWarps;
    double* all = all_sh[plain];
    if (tid == 0) {
      double c = 0.0;  // one after the other: the sums never decrease
      for (int i = 0; i < nws; i += kWarps) {
        double v[kWarps];
#pragma unroll
        for (int k = 0; k < kWarps; ++k) v[k] = all[i + k];
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          all[i + k] = c;
          c += v[k];
        }
      }
      all[nws] = c;
    }
    __syncthreads();
    const double total = all[nws];
    if (total > 0.0) {
      // below total whatever the uniform is, so some token exceeds it
      const double want = fmin(fmax(a.uniform(rows.y - 1), 0.0), 1.0 - 2.220446049250313e-16) * total;
      const double* ours = all + rank * kWarps;
      if (ours[0] <= want && ours[kWarps] > want) {  // this CTA's words hold it: a warp's share of them, an eighth of that
        int at = 0;
        while (ours[at + 1] <= want) ++at;
        const int wa = min(s.nw, at * per), wz = min(s.nw, wa + per), sub = (wz - wa + kWarps - 1) / kWarps;
        const double part = warp_left(min(wz, wa + warp * sub), min(wz, wa + (warp + 1) * sub), plain != 0);
        if (lane == 0) sub_sh[warp] = part;
        __syncthreads();
        if (warp == 0) {
          // (sums in another order may end a rounding before ``want``: then it is the last token with weight)
          double c = ours[at], c_last = c;
          int k = 0, last = 0;
          for (; k < kWarps; ++k) {
            if (sub_sh[k] > 0.0) last = k, c_last = c;
            if (c + sub_sh[k] > want) break;
            c += sub_sh[k];
          }
          if (k == kWarps) k = last, c = c_last;
          int tok = -1;
          const int wk = min(wz, wa + k * sub), we = min(wz, wk + sub);
          for (int wb = wk; wb < we; wb += 32) {
            double mine = 0.0, l[PER];
            const bool some_here = wb + lane < we && word_left(wb + lane, plain != 0, l);
            if (some_here)
#pragma unroll
              for (int j = 0; j < PER; ++j) mine += l[j];
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
      }
      break;
    }
    if (plain == 1 && rank == 0 && tid == 0) out[acc] = 0;  // no logit above -inf
  }
  if (rank == 0) finish();
}

// What the largest launch needs, once per device: the same values every time, so calls from several threads may meet here.
void allow_launches(int device) {
  static std::atomic<bool> done[64];
  if (device < 64 && done[device].load()) return;
  constexpr int kSmem = kMaxVocab * 4 / kMaxCluster + 64;
  static_assert(kSmem >= 44 * 1024 + 64);
  for (auto kern : {verify_rows_kernel<float>, verify_rows_kernel<bf16>, verify_draw_kernel<float>, verify_draw_kernel<bf16>}) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  }
  if (device < 64) done[device].store(true);
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
  // per row: cut; largest logit, acceptance; weights, tokens and number of listed tokens
  auto scratch = at::empty({R * (2 + kList + kList / 2) + (R + 1) / 2}, ids.options());
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
  a.kept_w = reinterpret_cast<double*>(scratch.data_ptr<int64_t>() + 2 * R);
  a.kept_tok = reinterpret_cast<int*>(a.kept_w + R * kList);
  a.kept_n = a.kept_tok + R * kList;
  a.err = err.data_ptr<int>();
  allow_launches(logits.get_device());
  auto stream = at::cuda::getCurrentCUDAStream();
  const bool wide = logits.scalar_type() == at::kFloat;
  const int64_t width = wide ? 4 : 2;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  // CTAs per row: as few as hold it in slices of 44 KB, four of which fit an SM; 8 while they all run at once (151936
  // tokens in bf16, 48 rows with a top_p: 50 against 53 us; 577 rows in 8 127, in 7 124 us) and for short rows while SMs
  // would idle; 16 (beyond the portable size) for rows that 8 would hold in larger slices
  auto cluster_for = [&](int64_t count) {
    int64_t n = (V * width + 44 * 1024 - 1) / (44 * 1024);
    if (n > 8) return (int64_t)kMaxCluster;
    if (n > 3 && count * 8 <= 4 * sms) return (int64_t)8;
    while (n < 8 && count * n * 2 <= sms) n = std::min<int64_t>(8, n * 2);
    return n;
  };
  auto run = [&](auto kern, int64_t count) {
    const int64_t n = cluster_for(count);
    const size_t smem = (size_t)(((V + n - 1) / n + 7) / 8 * 8 * width + 32);
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
