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

#include <algorithm>
#include <cmath>
#include <string>
#include <tuple>
#include <type_traits>

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
  int G;              // query heads of a KV head
  uint32_t g_magic;   // ceil(2^32 / G), 0 for G = 1
  float scale, softcap;
  int window;
  int* err;

  // (f / G, f % G): the high word of f ceil(2^32 / G) is the quotient as long as f G < 2^32
  NV_DEVICE int2 split(int f) const {
    const int t = g_magic == 0 ? f : (int)__umulhi((uint32_t)f, g_magic);
    return make_int2(t, f - t * G);
  }
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

// ------------------------------------------------------------------------------------------------ split kernels
// o = sum_i w_i O_i / sum_i w_i with w_i = 2^(lse_i - max lse): every part of the keys (a range of the prefix or of a
// sequence's own keys) is reduced by one CTA to a normalised fp32 row O_i and its log2-sum-exp, and a last kernel
// joins them.  Parts are written by every CTA, also by one whose range is empty (lse -inf), so nothing needs clearing.
constexpr int KT = 64;       // keys per tile
constexpr int kRows = 64;    // query rows (token, head of the group) per CTA of the mma.sync kernel
constexpr int kCuSmem = 1024;  // sequences whose cu_q fits the shared copy

struct SpPlan {
  int n_pre, pre_tiles, pre_row_tiles;  // prefix: key splits, tiles per split, row tiles
  int n_own, own_tiles, own_row_tiles;  // own keys: the same, per sequence
  int pre_slots;                        // parts of the prefix
  int tc;                               // the prefix is left to the tcgen05 kernel
  float* part_o;                        // [T, nq, pre_slots + n_own, hd]
  float* part_lse;                      // [T, nq, pre_slots + n_own]

  NV_DEVICE int slots() const { return pre_slots + n_own; }
};

// A page number as the tables give it, or page 0 and an error.
NV_DEVICE int sp_page(const SpArgs& a, int blk) {
  if (blk < 0 || blk >= a.num_blocks) {
    nvb::record_error(a.err, nvb::kErrBadArgument);
    return 0;
  }
  return blk;
}
// The page of tile ``tile`` (of ``keys`` keys) where the table has one.
NV_DEVICE int sp_table(const SpArgs& a, const int* pages, int n_pages, int tile, int keys) {
  const int at = (int)((long)tile * keys / a.block_size);
  return at < n_pages ? pages[at] : -1;
}

// cu_q in shared memory (global beyond kCuSmem sequences): the search for a row's sequence is then free of
// dependent global loads.
NV_DEVICE const int* stage_cu(const SpArgs& a, int* sh, int threads) {
  if (a.cu_q == nullptr || a.B >= kCuSmem) return a.cu_q;
  for (int i = threadIdx.x; i <= a.B; i += threads) sh[i] = a.cu_q[i];
  return sh;
}

// Position of query token t (-1: it sees no key, also for rows behind the last sequence or of a refused one).
NV_DEVICE int row_position(const SpArgs& a, const int* cu, int t, int P) {
  if (t >= a.T) return -1;
  int b = t, i = 0, n = 1;
  if (cu != nullptr) {
    b = seq_of(cu, a.B, t);
    const int lo = cu[b], hi = cu[b + 1];
    i = t - lo, n = hi - lo;
    if (lo < 0 || hi > a.T || t < lo || t >= hi || n > a.max_q) return -1;
  }
  const int ctx = a.ctx_lens[b];
  return a.ctx_ok(ctx, P) ? ctx - n + i : -1;
}

// One part: rows [row0, row0 + rows) of a (token, head) list against tiles [t0, t1) of the keys [klo, kend).
struct SpPart {
  int tok0, row0, rows;  // row r: token tok0 + (row0 + r) / G, head kvh * G + (row0 + r) % G
  int kvh, slot;
  int klo, kend, t0, t1;
  const int* pages;
  int n_pages;
  int page;  // in warp 0: the page of tile t0 + lane
};

// Four warps: RG groups of 16 rows times 4 / RG groups of 16 * RG keys of each tile.  S and O stay in registers
// (mma.sync m16n8k16), Q in registers up to head dim 128.
template <int HD, int STAGES, int RG>
__device__ void sp_part_mma(const SpArgs& a, const SpPlan& pl, const SpPart& p, const CUtensorMap* kmap,
                            const CUtensorMap* vmap, uint8_t* ring, uint64_t* bars, bf16* qs, const int* row_pos,
                            volatile int* abort_flag) {
  constexpr int TILE = KT * HD * 2;
  constexpr int KW = 16 * RG;  // keys of a warp
  constexpr int NB = KW / 8;
  constexpr int QP = HD + 8;
  constexpr bool kQRegs = HD <= 128;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c4 = lane & 3;
  const int rg = warp % RG, key0 = (warp / RG) * KW;
  const int G = a.G, nt = p.t1 - p.t0;
  int page = p.page;
  // Warp 0: the page of tile i, of which the lanes hold 32 at a time (a table look-up for each copy would come before it).
  auto page_of = [&](int i) {
    if (i >= 32 && (i & 31) == 0) page = sp_table(a, p.pages, p.n_pages, p.t0 + i + lane, KT);
    return __shfl_sync(0xffffffffu, page, i & 31);
  };
  auto issue = [&](int i, int pg) {
    const int st = i % STAGES, tok = (p.t0 + i) * KT;
    const int row = (sp_page(a, pg) * a.nkv + p.kvh) * a.block_size + tok % a.block_size;
    uint8_t* kd = ring + st * 2 * TILE;
    nvb::mbar_arrive_expect_tx(&bars[st], 2 * TILE);
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) {
      nvb::tma_load_2d(kd + j * KT * 128, kmap, &bars[st], j * 64, row);
      nvb::tma_load_2d(kd + TILE + j * KT * 128, vmap, &bars[st], j * 64, row);
    }
  };
  if (warp == 0)
    for (int i = 0; i < STAGES && i < nt; ++i) {
      const int pg = page_of(i);
      if (lane == 0) issue(i, pg);
    }
  auto q_row = [&](int r) {
    const int2 f = a.split(p.row0 + r);
    return a.q + (long)(p.tok0 + f.x) * a.q_tok + (long)(p.kvh * G + f.y) * a.q_head;
  };
  uint32_t qf[kQRegs ? HD / 16 : 1][4];
  if constexpr (kQRegs) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = rg * 16 + g + h * 8;
      const bf16* src = r < p.rows ? q_row(r) : nullptr;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        qf[kk][h] = src != nullptr ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 2 * c4) : 0u;
        qf[kk][h + 2] = src != nullptr ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8 + 2 * c4) : 0u;
      }
    }
  } else {
    for (int idx = tid; idx < 16 * RG * (HD / 8); idx += 128) {
      const int r = idx / (HD / 8), c = idx % (HD / 8);
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < p.rows) v = *reinterpret_cast<const uint4*>(q_row(r) + c * 8);
      *reinterpret_cast<uint4*>(qs + r * QP + c * 8) = v;
    }
    __syncthreads();
  }
  int rpos[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = rg * 16 + g + h * 8;
    rpos[h] = r < p.rows ? row_pos[r] : -1;
  }
  const int win = a.window > 0 ? a.window : 0x40000000;
  float o[HD / 8][4];
#pragma unroll
  for (int d = 0; d < HD / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  const float sl2 = a.scale * kLog2e;
  const int mi = lane >> 3, lr = lane & 7;
  bool aborted = false;
  for (int i = 0; i < nt; ++i) {
    const int st = i % STAGES;
    const bool ok = nvb::mbar_wait(&bars[st], (uint32_t)((i / STAGES) & 1), a.err, abort_flag);
    if (__syncthreads_or(!ok)) { aborted = true; break; }
    uint8_t* vt = ring + st * 2 * TILE + TILE;
    const uint32_t kb = nvb::smem_u32(ring + st * 2 * TILE), vb = kb + TILE;
    const int tok0 = (p.t0 + i) * KT;
    if (tok0 < p.klo || tok0 + KT > p.kend) {
      // keys outside the part may hold anything: their weight is 0, and 0 * NaN must not reach the sum
      const int lo = max(0, p.klo - tok0), hi = min(KT, p.kend - tok0);
      for (int idx = tid; idx < KT * (HD / 8); idx += 128) {
        const int r = idx / (HD / 8), c = idx % (HD / 8);
        if (r < lo || r >= hi)
          *reinterpret_cast<uint4*>(vt + (c >> 3) * (KT * 128) + nvb::swz128(r, c & 7)) = make_uint4(0, 0, 0, 0);
      }
      nvb::fence_proxy_async();  // before a later TMA copy into the same stage
      __syncthreads();
    }
    if (rg * 16 < p.rows) {
      float s[NB][4];
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t af[4];
        if constexpr (kQRegs) {
#pragma unroll
          for (int e = 0; e < 4; ++e) af[e] = qf[kk][e];
        } else {
          nvb::ldmatrix_x4(af[0], af[1], af[2], af[3],
                           nvb::smem_u32(qs) + ((rg * 16 + (lane & 15)) * QP + kk * 16 + (lane >> 4) * 8) * 2);
        }
#pragma unroll
        for (int np = 0; np < NB / 2; ++np) {
          const int key = key0 + np * 16 + lr + (mi >> 1) * 8, dim = kk * 16 + (mi & 1) * 8;
          uint32_t b0, b1, b2, b3;
          nvb::ldmatrix_x4(b0, b1, b2, b3, kb + (uint32_t)(dim >> 6) * (KT * 128) + nvb::swz128(key, (dim & 63) >> 3));
          nvb::mma_bf16_16816(s[2 * np], af, b0, b1);
          nvb::mma_bf16_16816(s[2 * np + 1], af, b2, b3);
        }
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1, key = tok0 + key0 + n * 8 + 2 * c4 + (e & 1);
          float x = a.softcap > 0.f ? sp_cap(s[n][e] * a.scale, a.softcap) * kLog2e : s[n][e] * sl2;
          if (key > rpos[h] || key < p.klo || key >= p.kend || key <= rpos[h] - win) x = -INFINITY;
          s[n][e] = x;
          mx[h] = fmaxf(mx[h], x);
        }
      float corr[2], rs[2] = {0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const float nm = fmaxf(m_run[h], mx[h]);
        corr[h] = nm == -INFINITY ? 1.f : exp2f(m_run[h] - nm);
        m_run[h] = nm;
      }
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1;
          const float w = m_run[h] == -INFINITY ? 0.f : exp2f(s[n][e] - m_run[h]);
          s[n][e] = w;
          rs[h] += w;
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) l_run[h] = l_run[h] * corr[h] + rs[h];
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        o[d][0] *= corr[0];
        o[d][1] *= corr[0];
        o[d][2] *= corr[1];
        o[d][3] *= corr[1];
      }
      // the weights are rounded to bf16 for the product (2^-8 of each, as everywhere in this engine); the
      // denominator sums them unrounded
#pragma unroll
      for (int ks = 0; ks < KW / 16; ++ks) {
        const uint32_t pa[4] = {nvb::pack_bf16x2(s[2 * ks][0], s[2 * ks][1]), nvb::pack_bf16x2(s[2 * ks][2], s[2 * ks][3]),
                                nvb::pack_bf16x2(s[2 * ks + 1][0], s[2 * ks + 1][1]),
                                nvb::pack_bf16x2(s[2 * ks + 1][2], s[2 * ks + 1][3])};
#pragma unroll
        for (int dp = 0; dp < HD / 16; ++dp) {
          const int key = key0 + ks * 16 + lr + (mi & 1) * 8, dim = dp * 16 + (mi >> 1) * 8;
          uint32_t b0, b1, b2, b3;
          nvb::ldmatrix_x4_trans(b0, b1, b2, b3,
                                 vb + (uint32_t)(dim >> 6) * (KT * 128) + nvb::swz128(key, (dim & 63) >> 3));
          nvb::mma_bf16_16816(o[2 * dp], pa, b0, b1);
          nvb::mma_bf16_16816(o[2 * dp + 1], pa, b2, b3);
        }
      }
    }
    __syncthreads();
    if (warp == 0 && i + STAGES < nt) {
      const int pg = page_of(i + STAGES);
      if (lane == 0) issue(i + STAGES, pg);
    }
  }
  if (aborted) {  // reported in the error word; drain the copies still in flight (bounded)
    if (tid == 0)
      for (int s = 0; s < STAGES; ++s) nvb::mbar_wait(&bars[s], 0, nullptr, nullptr);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
    l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
  }
  const int NS = pl.slots();
  auto slot_of = [&](int r) {
    const int2 f = a.split(p.row0 + r);
    return ((long)(p.tok0 + f.x) * a.nq + p.kvh * G + f.y) * NS + p.slot;
  };
  if constexpr (RG == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = rg * 16 + g + h * 8;
      if (r >= p.rows) continue;
      const long slot = slot_of(r);
      const float inv = l_run[h] > 0.f ? 1.f / l_run[h] : 0.f;
      float* dst = pl.part_o + slot * HD;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
        *reinterpret_cast<float2*>(dst + d * 8 + 2 * c4) = make_float2(o[d][2 * h] * inv, o[d][2 * h + 1] * inv);
      if (c4 == 0) pl.part_lse[slot] = l_run[h] > 0.f ? m_run[h] + log2f(l_run[h]) : -INFINITY;
    }
  } else {
    // join the key groups of a row group through shared memory (the ring is free: every tile was waited for)
    float* comb = reinterpret_cast<float*>(ring);  // [4 warps][16][HD]
    float* cm = comb + 4 * 16 * HD;                // [4][16]
    float* cl = cm + 64;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float2*>(comb + (warp * 16 + g + h * 8) * HD + d * 8 + 2 * c4) =
            make_float2(o[d][2 * h], o[d][2 * h + 1]);
    if (c4 == 0)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        cm[warp * 16 + g + h * 8] = m_run[h];
        cl[warp * 16 + g + h * 8] = l_run[h];
      }
    __syncthreads();
    for (int idx = tid; idx < p.rows * (HD / 4); idx += 128) {
      const int r = idx / (HD / 4), d = (idx % (HD / 4)) * 4;
      const int w0 = r >> 4, rr = r & 15;  // warps w0, w0 + RG, ... hold the row
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4 / RG; ++w) M = fmaxf(M, cm[(w0 + w * RG) * 16 + rr]);
      float L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      if (M != -INFINITY) {
#pragma unroll
        for (int w = 0; w < 4 / RG; ++w) {
          const int at = (w0 + w * RG) * 16 + rr;
          const float f = exp2f(cm[at] - M);
          const float4 v = *reinterpret_cast<const float4*>(comb + at * HD + d);
          L += cl[at] * f;
          acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
        }
      }
      const float inv = L > 0.f ? 1.f / L : 0.f;
      const long slot = slot_of(r);
      *reinterpret_cast<float4*>(pl.part_o + slot * HD + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (d == 0) pl.part_lse[slot] = L > 0.f ? M + log2f(L) : -INFINITY;
    }
  }
}

template <int HD, int STAGES>
constexpr size_t sp_mma_smem() {
  return 1024 + STAGES * 2 * KT * HD * 2 + (HD <= 128 ? 0 : kRows * (HD + 8) * 2) + 64;
}

// Grid: the parts of the prefix (split fastest, then KV head, then row tile), then those of the sequences' own keys
// (split, KV head, row tile, sequence).  K/V tiles of 64 keys come through TMA into a ring of STAGES; bound by the
// bytes of the cache as long as a tile serves few rows.
template <int HD, int STAGES, int MAX_RG>
__device__ __forceinline__ void sp_mma_part(const CUtensorMap& kmap, const CUtensorMap& vmap, const SpArgs& a,
                                            const SpPlan& pl) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  bf16* qs = reinterpret_cast<bf16*>(ring + STAGES * 2 * KT * HD * 2);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(qs) + (HD <= 128 ? 0 : kRows * (HD + 8) * 2));
  __shared__ int abort_flag, cu_sh[kCuSmem + 1], row_pos[kRows], pos_lo, pos_hi;
  const int tid = threadIdx.x;
  const int G = a.G, P = a.prefix_len();
  const bool p_ok = a.prefix_ok(P);
  SpPart p{};
  int bid = blockIdx.x;
  const int n_prefix = pl.tc ? 0 : pl.n_pre * a.nkv * pl.pre_row_tiles;
  const bool is_prefix = bid < n_prefix;
  if (tid == 0) {
    abort_flag = 0;
    pos_lo = 0x7fffffff;
    pos_hi = -1;
    for (int s = 0; s < STAGES; ++s) nvb::mbar_init(&bars[s], 1);
    nvb::fence_mbar_init();
    nvb::tma_prefetch_desc(&kmap);
    nvb::tma_prefetch_desc(&vmap);
  }
  if (is_prefix) {
    const int split = bid % pl.n_pre;
    bid /= pl.n_pre;
    p.kvh = bid % a.nkv;
    p.row0 = (bid / a.nkv) * kRows;
    p.rows = min(kRows, a.T * G - p.row0);
    p.slot = split;
    p.kend = p_ok ? P : 0;
    p.t0 = split * pl.pre_tiles;
    p.t1 = p.t0 + pl.pre_tiles;
    p.pages = a.prefix_blocks;
    p.n_pages = a.n_prefix_blocks;
    if (tid < 32) p.page = sp_table(a, p.pages, p.n_pages, p.t0 + tid, KT);
    const int* cu = stage_cu(a, cu_sh, 128);
    __syncthreads();
    if (tid < kRows && tid < p.rows) {
      const int pos = row_position(a, cu, a.split(p.row0 + tid).x, P);
      row_pos[tid] = pos;
      if (pos >= 0) {
        atomicMin(&pos_lo, pos);
        atomicMax(&pos_hi, pos);
      }
    }
  } else {
    bid -= n_prefix;
    const int split = bid % pl.n_own;
    bid /= pl.n_own;
    p.kvh = bid % a.nkv;
    bid /= a.nkv;
    const int b = bid / pl.own_row_tiles;
    p.t0 = max(0, P) / KT + split * pl.own_tiles;
    p.pages = a.block_tables + b * a.bt_stride;
    p.n_pages = a.bt_width;
    if (tid < 32) p.page = sp_table(a, p.pages, p.n_pages, p.t0 + tid, KT);  // (while the lengths are on their way)
    const int2 tk = a.tokens(b);
    const int ctx = a.ctx_lens[b], n = tk.y - tk.x;
    if (n < 0 || !p_ok || !a.ctx_ok(ctx, P)) {  // reported; the sequence's rows are undefined
      if (tid == 0) nvb::record_error(a.err, nvb::kErrBadArgument);
      return;
    }
    p.tok0 = tk.x;
    p.row0 = (bid % pl.own_row_tiles) * kRows;
    p.rows = min(kRows, n * G - p.row0);
    if (p.rows <= 0) return;
    p.slot = pl.pre_slots + split;
    p.klo = P;
    p.kend = ctx;
    p.t1 = p.t0 + pl.own_tiles;
    __syncthreads();
    if (tid < p.rows) {
      const int pos = ctx - n + a.split(p.row0 + tid).x;
      row_pos[tid] = pos;
      if (tid == 0) pos_lo = pos;
      if (tid == p.rows - 1) pos_hi = pos;
    }
  }
  __syncthreads();
  if (is_prefix && !p_ok && tid == 0) nvb::record_error(a.err, nvb::kErrBadArgument);
  // only tiles that some row sees
  p.kend = min(p.kend, pos_hi + 1);
  p.t1 = p.kend > p.klo ? min(p.t1, (p.kend + KT - 1) / KT) : p.t0;
  if (a.window > 0 && pos_lo != 0x7fffffff && max(0, pos_lo - a.window + 1) / KT > p.t0) {
    p.t0 = max(0, pos_lo - a.window + 1) / KT;
    if (tid < 32) p.page = sp_table(a, p.pages, p.n_pages, p.t0 + tid, KT);
  }
  if (p.t0 >= p.t1) {
    const int NS = pl.slots();
    if (tid < p.rows) {
      const int2 f = a.split(p.row0 + tid);
      pl.part_lse[((long)(p.tok0 + f.x) * a.nq + p.kvh * G + f.y) * NS + p.slot] = -INFINITY;
    }
    return;
  }
  if (MAX_RG == 1 || p.rows <= 16) sp_part_mma<HD, STAGES, 1>(a, pl, p, &kmap, &vmap, ring, bars, qs, row_pos, &abort_flag);
  else if (MAX_RG == 2 || p.rows <= 32)
    sp_part_mma<HD, STAGES, MAX_RG == 1 ? 1 : 2>(a, pl, p, &kmap, &vmap, ring, bars, qs, row_pos, &abort_flag);
  else sp_part_mma<HD, STAGES, MAX_RG>(a, pl, p, &kmap, &vmap, ring, bars, qs, row_pos, &abort_flag);
}

// The own keys (and the prefix where no tcgen05 kernel takes it) on mma.sync: a part has at most 64 rows, usually the few
// of one sequence, and reads its keys once, so it is bound by the bytes of K and V.  Measured: 128 sequences of 64 to 1024
// own keys, 8 KV heads, 285 MB: 56 us (5.1 TB/s), beside the prefix on a third of the SMs 72 us.
// ``MAX_RG``: row groups of the largest part.  A CTA spends some 3 us on either side of its stream of tiles, which the
// others of its SM fill: three of them where the registers allow it (parts of up to 32 rows, head dim up to 128).
template <int HD, int STAGES, int MAX_RG>
__global__ void __launch_bounds__(128, HD <= 128 && MAX_RG <= 2 ? 3 : 1) sp_mma_kernel(const __grid_constant__ CUtensorMap kmap,
                                                     const __grid_constant__ CUtensorMap vmap, const SpArgs a,
                                                     const SpPlan pl) {
  // After the tcgen05 kernel nothing here depends on its results: the parts run beside it, on the SMs that it leaves
  // free.  That kernel has waited for its own predecessor before it let this one start.  The last CTA waits for it at
  // the end, so that the join, which waits for this kernel, comes after both.
  if (!pl.tc) nvb::pdl_wait();
  nvb::pdl_trigger();
  sp_mma_part<HD, STAGES, MAX_RG>(kmap, vmap, a, pl);
  if (pl.tc && blockIdx.x == gridDim.x - 1) nvb::pdl_wait();
}

// One warp per (token, head): joins the parts.  Bound by the latency of two dependent reads, 6 to 11 us.
template <int HD>
__global__ void __launch_bounds__(128) sp_join_kernel(SpArgs a, SpPlan pl) {
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, NS = pl.slots();
  const int t = (int)((uint32_t)row / (uint32_t)a.nq), h = (int)((uint32_t)row % (uint32_t)a.nq);
  const float* lse = pl.part_lse + row * NS;
  const float* po = pl.part_o + row * NS * HD;
  nvb::pdl_wait();
  nvb::pdl_trigger();
  if (row >= (long)a.T * a.nq) return;
  float M = -INFINITY;
  for (int s = lane; s < NS; s += 32) M = fmaxf(M, lse[s]);
  if (a.cu_q != nullptr && (t < a.cu_q[0] || t >= a.cu_q[a.B])) return;  // a row behind the last sequence
  M = nvb::warp_max(M);
  constexpr int PER = HD / 32;  // 2, 4 or 8 values per lane
  float acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
  float den = 0.f;
  if (M != -INFINITY)
    for (int s0 = 0; s0 < NS; s0 += 32) {
      const float w = s0 + lane < NS ? exp2f(lse[s0 + lane] - M) : 0.f;
      den += w;
      unsigned left = __ballot_sync(0xffffffffu, w > 0.f);
      while (left != 0) {  // four parts at a time: their loads do not wait for one another
        int at[4];
        float ws[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          at[k] = left != 0 ? __ffs(left) - 1 : (k > 0 ? at[0] : 0);
          ws[k] = __shfl_sync(0xffffffffu, w, at[k]);
          if (left == 0) ws[k] = 0.f;
          left &= left - 1;
        }
        float2 v[4][PER / 2];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < PER / 2; ++i)
            v[k][i] = *reinterpret_cast<const float2*>(po + (long)(s0 + at[k]) * HD + lane * PER + 2 * i);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int i = 0; i < PER / 2; ++i) {
            acc[2 * i] += ws[k] * v[k][i].x;
            acc[2 * i + 1] += ws[k] * v[k][i].y;
          }
      }
    }
  den = nvb::warp_sum(den);
  const float inv = den > 0.f ? 1.f / den : 0.f;
  bf16* dst = a.out + t * a.o_tok + h * a.o_head + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; i += 2)
    *reinterpret_cast<uint32_t*>(dst + i) = nvb::pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
}

#include "shared_prefix_tc.cuh"

template <int HD, int STAGES, int MAX_RG>
int launch_split(const SpArgs& a, const SpPlan& pl, const void* kc, const void* vc, cudaStream_t stream) {
  int launches = 1;
  const uint64_t rows = (uint64_t)a.num_blocks * a.nkv * a.block_size;
  const CUtensorMap km = nvb::make_tmap_2d_bf16(kc, rows, HD, HD, KT);
  const CUtensorMap vm = nvb::make_tmap_2d_bf16(vc, rows, HD, HD, KT);
  auto kern = sp_mma_kernel<HD, STAGES, MAX_RG>;
  constexpr size_t sm = sp_mma_smem<HD, STAGES>();
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
  if constexpr (HD <= 128) {
    if (pl.tc) {
      launch_tc<HD>(a, pl, kc, vc, stream);
      ++launches;
    }
  }
  const unsigned grid = (unsigned)((pl.tc ? 0 : pl.n_pre * a.nkv * pl.pre_row_tiles) +
                                   pl.n_own * a.nkv * pl.own_row_tiles * a.B);
  if (grid > 0) ++launches;
  if (grid > 0) C10_CUDA_CHECK(nvb::launch(kern, dim3(grid), dim3(128), sm, stream, km, vm, a, pl));
  C10_CUDA_CHECK(nvb::launch(sp_join_kernel<HD>, dim3((unsigned)(((long)a.T * a.nq + 3) / 4)), dim3(128), 0, stream, a, pl));
  return launches;
}

// Tiles per split so that ``groups`` independent row groups over ``tiles`` key tiles make about ``ctas`` CTAs, with at
// most 32 splits.
void split_keys(long groups, int tiles, long ctas, int* n, int* per) {
  *per = (int)std::max<long>(1, std::min<long>(16, groups * tiles / std::max<long>(1, ctas)));
  *per = std::max(*per, (tiles + 31) / 32);
  *n = (tiles + *per - 1) / *per;
}

// How many splits the tcgen05 kernel takes of the prefix.  Its CTAs have an SM each to themselves and the own keys' kernel
// runs on the others meanwhile, so the rule looks for the least time of the two together: a prefix CTA takes some 5 us and
// 1.7 us for every key tile (two tiles when both its row tiles are the same rows); the own keys stream at 6 TB/s, which
// two thirds of the SMs still reach; a split's parts are written and read again at some 1.3 TB/s.  (Measured with 1, 2, 3,
// 4, 5, 6, 8 splits: 32 sequences on 2048 keys 30, 23, 22, 21, 21, 23, 26 us; 128 on 8192 keys 143, 82, 72, 77, 81, 85,
// 91 us; 64 with drafts on 4096 keys 83, 51, 41, 49, 48, 51, 57 us; 96 on 16000 keys, head dim 64, 238, 127, 90, 73, 61,
// 61, 67 us.  Taken are 4, 3, 3 and 6.)
void split_prefix(int groups, int tiles, bool twice, double own_bytes, double part_bytes, int sms, int* n, int* per) {
  const double own_us = own_bytes / 6.0e6;
  double best = 1e30;
  for (int splits = 1; splits <= tiles && (splits == 1 || (long)splits * groups <= sms); ++splits) {
    const int each = (tiles + splits - 1) / splits;
    const double waves = std::ceil((double)splits * groups / sms);
    const double tc = waves * (5.0 + 1.7 * (twice ? (each + 1) / 2 : each));
    const double share = std::min(1.0, 1.5 * std::max(0, sms - splits * groups) / sms);  // of the stream, meanwhile
    const double total = (own_us <= share * tc ? tc : tc + (own_us - share * tc)) + splits * part_bytes / 1.3e6;
    if (total < best) {
      best = total;
      *n = splits;
      *per = each;
    }
  }
  *n = (tiles + *per - 1) / *per;
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
  TORCH_CHECK(max_len < (int64_t(1) << 30) && T * nq * (nq / nkv) < (int64_t(1) << 32) && T * nq < (int64_t(1) << 30) && window < (int64_t(1) << 30),
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
  a.G = (int)(nq / nkv);
  a.g_magic = a.G == 1 ? 0u : (uint32_t)(((uint64_t(1) << 32) + a.G - 1) / a.G);
  a.err = err.data_ptr<int>();
  auto stream = at::cuda::getCurrentCUDAStream();
  if (hd != 64 && hd != 128 && hd != 256) {
    const long warps = (long)T * nq;
    C10_CUDA_CHECK(nvb::launch(sp_generic_kernel, dim3((unsigned)((warps + 3) / 4)), dim3(128), 0, stream, a,
                               reinterpret_cast<const bf16*>(k_cache.data_ptr()),
                               reinterpret_cast<const bf16*>(v_cache.data_ptr())));
    return {out, 1};
  }
  const int G = a.G, sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int64_t pre_bound = prefix_len_dev.has_value() ? prefix_blocks.numel() * bs : prefix_len;
  const int64_t pre_keys = std::min<int64_t>(pre_bound, max_len);
  const int own_tiles = (int)std::max<int64_t>(0, (max_len + KT - 1) / KT - (prefix_len_dev.has_value() ? 0 : prefix_len / KT));
  SpPlan pl{};
  const int64_t rows = T * G;
  pl.tc = pre_keys > 0 && hd <= 128 && bs % 128 == 0 && rows > 64;
  if (pl.tc) {
    pl.pre_row_tiles = (int)((rows + 255) / 256);
    // half of the keys that the bound leaves to the sequences, on average
    const double own_bytes = 2.0 * (double)(max_len - pre_keys) * (double)(B * nkv * hd);
    split_prefix((int)(nkv * pl.pre_row_tiles), (int)((pre_keys + 127) / 128), rows <= 128, own_bytes,
                 8.0 * (double)(T * nq * hd) * (rows <= 128 ? 2 : 1), sms, &pl.n_pre, &pl.pre_tiles);
    pl.pre_slots = 2 * pl.n_pre;
  } else {
    pl.pre_row_tiles = (int)((rows + kRows - 1) / kRows);
    split_keys((long)nkv * pl.pre_row_tiles, (int)((pre_keys + KT - 1) / KT), 2 * sms, &pl.n_pre, &pl.pre_tiles);
    pl.pre_slots = pl.n_pre;
  }
  pl.own_row_tiles = (int)((std::min(max_q, T) * G + kRows - 1) / kRows);
  // one part for each SM: a part costs some microseconds beside its tiles (head dim 256, 64 sequences with 1 to 700 own
  // keys: 28 us with four for each, 21.6 us with one; head dim 128, 32 sequences: 23 and 21.7 us)
  split_keys((long)nkv * B * pl.own_row_tiles, own_tiles, sms, &pl.n_own, &pl.own_tiles);
  const int64_t parts = T * nq * (pl.pre_slots + pl.n_own);
  auto scratch = at::empty({parts * (hd + 1)}, q.options().dtype(at::kFloat));
  pl.part_o = scratch.data_ptr<float>();
  pl.part_lse = pl.part_o + parts * hd;
  const void *kp = k_cache.data_ptr(), *vp = v_cache.data_ptr();
  // rows of the largest part, and K/V in flight: 64 KB a CTA where three share an SM, 96 KB else
  const int64_t part_rows = std::max<int64_t>(std::min<int64_t>(max_q, T) * G, pl.tc ? 0 : rows);
  auto launch = [&](auto hd_, auto few, auto many) {
    constexpr int HD = decltype(hd_)::value, FEW = decltype(few)::value, MANY = decltype(many)::value;
    return part_rows <= 16   ? launch_split<HD, FEW, 1>(a, pl, kp, vp, stream)
           : part_rows <= 32 ? launch_split<HD, FEW, 2>(a, pl, kp, vp, stream)
                             : launch_split<HD, MANY, 4>(a, pl, kp, vp, stream);
  };
#define SP_INT(N) std::integral_constant<int, N>()
  const int launches = hd == 64    ? launch(SP_INT(64), SP_INT(4), SP_INT(4))
                       : hd == 128 ? launch(SP_INT(128), SP_INT(2), SP_INT(3))
                                   : launch(SP_INT(256), SP_INT(2), SP_INT(2));
#undef SP_INT
  return {out, launches};
}
