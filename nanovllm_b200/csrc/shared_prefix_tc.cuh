// The prefix's part of shared-prefix attention on the 5th-generation tensor cores.  Included by shared_prefix.cu.
//
// All query rows (token, head of the GQA group) of the batch stand against the same keys, so they fill MMA tiles of 128
// rows whatever sequence they come from.  One CTA per (range of keys, KV head, 256 rows) works on two tiles at once:
// while the softmax threads of one turn its scores into weights, the tensor cores run the other's products.
//   S_q = Q_q K^T    operands in shared memory, fp32 scores in tensor memory (128 columns per tile)
//   P_q = 2^(S - m)  one thread per row: scores from tensor memory, 32 columns at a time, P back as bf16 (rounded once,
//                    2^-9 of a weight; sums take the 32 bits) over columns that have been read
//   O_q += P_q V     A = P from tensor memory, B = V in shared memory, fp32 O in tensor memory
// With more than 128 rows the two tiles are rows [0, 128) and [128, 256) against every key tile; with fewer, both are
// the same rows, one against the even key tiles of the range, the other against the odd ones, and each writes a part.
// The maximum in use moves (and O, l are rescaled) only when a row's maximum grows by more than 2^8: weights stay
// below 2^8 and O / l is exact all the same.  Both products of a tile take as long as its exponentials (head dim 128:
// 1024 clocks each), so the kernel is bound by either pipe at best.  Measured: a step of both tiles takes 3400 clocks and
// a CTA some 5 us beside its steps; 128 rows x 4 heads against 8192 keys 57 us in 48 CTAs of 22 tiles, 32 x 4 against
// 2048 keys 15 us.
//
// Warps: 0 / 3 copy K / V tiles (TMA), 1 issues the MMAs, 2 clears the V rows behind the prefix, 4-7 and 8-11 are the
// softmax threads of the two tiles.  Every wait is bounded.
#pragma once

template <int HD>
struct SpTc {
  static constexpr int BN = 128;
  static constexpr int KS = HD == 64 ? 4 : 3, VS = HD == 64 ? 4 : 2;
  static constexpr int KBOX = BN * 128;           // 64 dims of a K or V tile, bytes
  static constexpr int KTILE = (HD / 64) * KBOX;
  static constexpr int QBOX = 128 * 128;          // 64 dims of 128 query rows
  static constexpr int QTILE = (HD / 64) * QBOX;
  static constexpr uint32_t O_COL = 2 * BN;       // tensor memory: S of both tiles, then O of both
  static_assert(O_COL + 2 * HD <= 512, "tensor memory plan");
  static constexpr int kBars = 2 * KS + 2 * VS + 7;
  static constexpr size_t smem() { return 1024 + 2 * QTILE + (size_t)(KS + VS) * KTILE + kBars * 8; }
};

NV_DEVICE void tc_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
NV_DEVICE void tc_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
NV_DEVICE void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
NV_DEVICE void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D(tmem) (+)= A(tmem) B(smem), bf16 operands
NV_DEVICE void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// True in one lane of a converged warp, always the same one.  The MMAs stand in a branch on it and not on lane == 0:
// measured beside busy softmax warps, an issue then costs 85-100 cycles against 170 (64 either way on a quiet SM).
NV_DEVICE bool tc_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}
// V as an MN-major operand: rows (keys) along K in 8-row swizzle atoms, 64-dim boxes ``mn_stride`` bytes apart along N.
NV_DEVICE uint64_t tc_desc_v(uint32_t addr, uint32_t mn_stride) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((mn_stride >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)2u << 61;
  return d;
}
// Bounded wait that looks at the barrier a few times before it reads the clock (which takes longer than most waits).
NV_DEVICE bool tc_wait(uint64_t* bar, uint32_t parity, int* err, volatile int* abort_flag) {
#pragma unroll 1
  for (int i = 0; i < 32; ++i)
    if (nvb::mbar_try_wait(bar, parity)) return true;
  return nvb::mbar_wait(bar, parity, err, abort_flag);
}

// two fp32 values in one register pair, and operations on both at once
NV_DEVICE uint64_t pack2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
NV_DEVICE void unpack2(uint64_t d, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d)); }
NV_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
NV_DEVICE uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^v of two values on the FMA pipe, for a part of the weights: the special-function unit gives 16 a clock and SM, which
// for a whole tile is as long as the tile's products.  v = n + f with n the nearest integer (from the low bits of
// v + 1.5 * 2^23), 2^f by a polynomial of degree 4 fitted to the relative error on [-1/2, 1/2] (2.7e-6, far below the
// bf16 that the weight is rounded to), n added to the exponent.  Below -126 the result is 2^-126 instead of less.
NV_DEVICE void exp2_poly2(uint64_t v, float& p0, float& p1) {
  float x0, x1;
  unpack2(v, x0, x1);
  v = pack2(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t magic = pack2(12582912.f, 12582912.f), back = pack2(-12582912.f, -12582912.f);
  const uint64_t n = add2(v, magic);
  const uint64_t f = fma2(add2(n, back), pack2(-1.f, -1.f), v);
  uint64_t y = fma2(f, pack2(0.00957010221f, 0.00957010221f), pack2(0.0559178628f, 0.0559178628f));
  y = fma2(f, y, pack2(0.240247443f, 0.240247443f));
  y = fma2(f, y, pack2(0.693121791f, 0.693121791f));
  y = fma2(f, y, pack2(0.999999285f, 0.999999285f));
  float n0, n1, y0, y1;
  unpack2(n, n0, n1);
  unpack2(y, y0, y1);
  p0 = __int_as_float((__float_as_int(n0) << 23) + __float_as_int(y0));
  p1 = __int_as_float((__float_as_int(n1) << 23) + __float_as_int(y1));
}

// Sequence of the warp's first token by a 32-way search, then each lane walks on to its own token (consecutive tokens
// of a warp lie in the same or the next sequences).
NV_DEVICE int warp_row_position(const SpArgs& a, int t_first, int t, int P) {
  if (a.cu_q == nullptr) return row_position(a, nullptr, t, P);
  const int lane = threadIdx.x & 31;
  int lo = 0, len = a.B;
  while (len > 1) {  // cu_q[lo] <= t_first; the answer lies in [lo, lo + len)
    const int step = (len + 31) / 32, at = lo + lane * step;
    const bool below = at < lo + len && a.cu_q[at] <= t_first;
    const int n = __popc(__ballot_sync(0xffffffffu, below));
    const int skip = max(0, n - 1) * step;
    lo += skip;
    len = min(step, len - skip);
  }
  if (t >= a.T) return -1;
  int b = lo;
  while (b + 1 < a.B && a.cu_q[b + 1] <= t) ++b;
  const int c0 = a.cu_q[b], c1 = a.cu_q[b + 1];
  if (c0 < 0 || c1 > a.T || t < c0 || t >= c1 || c1 - c0 > a.max_q) return -1;
  const int ctx = a.ctx_lens[b];
  return a.ctx_ok(ctx, P) ? ctx - (c1 - c0) + (t - c0) : -1;
}

template <int HD>
__global__ void __launch_bounds__(384, 1) sp_tc_kernel(const __grid_constant__ CUtensorMap kmap,
                                                       const __grid_constant__ CUtensorMap vmap, const SpArgs a,
                                                       const SpPlan pl) {
  using C = SpTc<HD>;
  constexpr int BN = C::BN, KS = C::KS, VS = C::VS;
  constexpr uint32_t IDESC_S = nvb::idesc_bf16_f32(128, BN);
  constexpr uint32_t IDESC_PV = nvb::idesc_bf16_f32(128, HD) | (1u << 16);  // V is MN-major
  extern __shared__ uint8_t smem_raw[];
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* kring = qs + 2 * C::QTILE;
  uint8_t* vring = kring + (size_t)KS * C::KTILE;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(vring + (size_t)VS * C::KTILE);
  uint64_t* k_free = k_full + KS;
  uint64_t* v_full = k_free + KS;
  uint64_t* v_free = v_full + VS;
  uint64_t* s_full = v_free + VS;  // [2] scores of a tile
  uint64_t* p_full = s_full + 2;   // [2] its weights
  uint64_t* o_done = p_full + 2;   // [2] its product with V
  uint64_t* v_clear = o_done + 2;    // the last V tile without what lies behind the prefix
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_flag, pos_lo, pos_hi;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    abort_flag = 0;
    pos_lo = 0x7fffffff;
    pos_hi = -1;
    for (int s = 0; s < KS; ++s) {
      nvb::mbar_init(&k_full[s], 1);
      nvb::mbar_init(&k_free[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      nvb::mbar_init(&v_full[s], 1);
      nvb::mbar_init(&v_free[s], 1);
    }
    for (int q = 0; q < 2; ++q) {
      nvb::mbar_init(&s_full[q], 1);
      nvb::mbar_init(&p_full[q], 4);
      nvb::mbar_init(&o_done[q], 1);
    }
    nvb::mbar_init(v_clear, 1);
    nvb::fence_mbar_init();
    nvb::tma_prefetch_desc(&kmap);
    nvb::tma_prefetch_desc(&vmap);
  }
  if (warp == 1) {
    nvb::tmem_alloc(&tmem_base_sh, 512);
    nvb::tmem_relinquish();
  }
  nvb::pdl_wait();
  nvb::pdl_trigger();

  const int G = a.G, P = a.prefix_len();
  int bid = blockIdx.x;
  const int split = bid % pl.n_pre;
  bid /= pl.n_pre;
  const int kvh = bid % a.nkv, row0 = (bid / a.nkv) * 256;
  const int rows = min(256, a.T * G - row0);
  const bool twice = rows <= 128;  // both tiles are the same rows
  const int kend = a.prefix_ok(P) ? P : 0;
  int t0 = split * pl.pre_tiles;
  const int t1 = min(t0 + pl.pre_tiles, (kend + BN - 1) / BN);
  // one K or V tile into its ring
  auto copy = [&](bool is_k, int i, int pg) {
    const int s = i % (is_k ? KS : VS), tok = (t0 + i) * BN;
    const int row = (sp_page(a, pg) * a.nkv + kvh) * a.block_size + tok % a.block_size;
    uint8_t* dst = (is_k ? kring : vring) + (size_t)s * C::KTILE;
    uint64_t* bar = is_k ? &k_full[s] : &v_full[s];
    nvb::mbar_arrive_expect_tx(bar, C::KTILE);
#pragma unroll
    for (int j = 0; j < HD / 64; ++j) nvb::tma_load_2d(dst + j * C::KBOX, is_k ? &kmap : &vmap, bar, j * 64, row);
  };
  // the copying warps' lanes hold the pages of 32 tiles
  int page = -1;
  auto page_of = [&](int i) {
    if (i > 0 && (i & 31) == 0) page = sp_table(a, a.prefix_blocks, a.n_prefix_blocks, t0 + i + lane, BN);
    return __shfl_sync(0xffffffffu, page, i & 31);
  };
  const bool early = a.window <= 0;  // the first key tile is known before the rows' positions are
  if (early && (warp == 0 || warp == 3)) page = sp_table(a, a.prefix_blocks, a.n_prefix_blocks, t0 + lane, BN);
  if (warp == 0) {
    if (lane == 0 && !a.prefix_ok(P)) nvb::record_error(a.err, nvb::kErrBadArgument);
    if (early)
      for (int i = 0; i < max(KS, VS) && i < t1 - t0; ++i) {
        const int pg = page_of(i);
        if (lane == 0 && i < KS) copy(true, i, pg);
        if (lane == 0 && i < VS) copy(false, i, pg);
      }
  }
  // The softmax threads load the query rows, into the swizzled layout that the MMA reads (zeros behind the list), and
  // find the rows' positions.
  const int tile = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;  // warps 4-11
  const int rr = row0 + (twice ? 0 : tile * 128) + r;             // row of the list
  int pos = -1;                                                   // no key seen
  if (warp >= 4) {
    if (!(twice && tile == 1)) {
      constexpr int CH = HD / 8, STEP = 128 / CH;  // 16-byte chunks of a row; rows that the 128 threads load at once
      const int c = tid % CH, first = (tid & 127) / CH;
      uint8_t* qt = qs + tile * C::QTILE + (c >> 3) * C::QBOX;
      const bf16* src = a.q + (long)kvh * G * a.q_head + c * 8;
      uint4 v[CH];
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int f = row0 + tile * 128 + first + k * STEP;
        v[k] = make_uint4(0, 0, 0, 0);
        const int2 tg = a.split(f);
        if (f < row0 + rows) v[k] = *reinterpret_cast<const uint4*>(src + (long)tg.x * a.q_tok + (long)tg.y * a.q_head);
      }
#pragma unroll
      for (int k = 0; k < CH; ++k)
        *reinterpret_cast<uint4*>(qt + nvb::swz128(first + k * STEP, c & 7)) = v[k];
      nvb::fence_proxy_async();
    }
    const int first = row0 + (twice ? 0 : tile * 128) + (warp & 3) * 32;
    if (first < row0 + rows) {
      pos = warp_row_position(a, a.split(first).x, a.split(rr).x, P);
      if (rr >= row0 + rows) pos = -1;
    }
    if (!early) {
      const int lo = __reduce_min_sync(0xffffffffu, pos < 0 ? 0x7fffffff : pos);
      const int hi = __reduce_max_sync(0xffffffffu, pos);
      if (lane == 0 && hi >= 0) {
        atomicMin(&pos_lo, lo);
        atomicMax(&pos_hi, hi);
      }
    }
  }
  nvb::tc_fence_before();
  __syncthreads();
  nvb::tc_fence_after();
  const uint32_t tmem = tmem_base_sh;
  // with a window: only the key tiles that some row sees
  if (!early) t0 = pos_hi < 0 ? t1 : max(t0, max(0, pos_lo - a.window + 1) / BN);
  const int nt = max(0, t1 - t0);
  // step j of tile q works on key tile t0 + j, or t0 + 2 j + q
  const int stride = twice ? 2 : 1;
  const int steps0 = twice ? (nt + 1) / 2 : nt, steps1 = twice ? nt / 2 : nt;
  const bool clear = nt > 0 && (t0 + nt) * BN > kend;  // the last tile ends behind the prefix

  // registers: launched with 168 a thread (64512 in all); 128 * 88 + 256 * 208 is the same sum
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0 || warp == 3) {
    // ---------------------------------------------------------------- copies
    const bool is_k = warp == 0;
    const int NS = is_k ? KS : VS;
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* freeb = is_k ? k_free : v_free;
    if (!early) page = sp_table(a, a.prefix_blocks, a.n_prefix_blocks, t0 + lane, BN);
    int i = early ? min(NS, nt) : 0;
    bool ok = true;
    for (; i < nt; ++i) {
      const int pg = page_of(i);
      if (i >= NS && !__all_sync(0xffffffffu, tc_wait(&freeb[i % NS], ((i / NS) & 1) ^ 1, a.err, &abort_flag))) {
        ok = false;
        break;
      }
      if (lane == 0) copy(is_k, i, pg);
      __syncwarp();
    }
    if (!ok && lane == 0)  // bounded drain of copies that may still be landing
      for (int j = (i > NS ? i - NS : 0); j < i; ++j) tc_wait(&full[j % NS], (j / NS) & 1, nullptr, nullptr);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issue
    // descriptors differ from these in the start address alone (16-byte units in the low bits)
    const uint64_t q_desc = nvb::sdesc_kmajor_sw128(nvb::smem_u32(qs)), k_desc = nvb::sdesc_kmajor_sw128(nvb::smem_u32(kring));
    const uint64_t v_desc = tc_desc_v(nvb::smem_u32(vring), C::KBOX);
    auto wait = [&](uint64_t* bar, int phase) {
      return __all_sync(0xffffffffu, tc_wait(bar, (uint32_t)(phase & 1), a.err, &abort_flag));
    };
    // scores of Q tile q against key tile i
    auto issue_s = [&](int q, int i, bool last_use) {
      const uint64_t kd = k_desc + (uint32_t)(i % KS) * (C::KTILE >> 4);
      const uint64_t qd = q_desc + (uint32_t)(twice ? 0 : q) * (C::QTILE >> 4);
      const uint32_t d = tmem + (uint32_t)q * BN;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        nvb::tc_mma_f16(d, qd + ((kk >> 2) * C::QBOX + (kk & 3) * 32) / 16,
                  kd + ((kk >> 2) * C::KBOX + (kk & 3) * 32) / 16, IDESC_S, kk > 0 ? 1u : 0u);
      nvb::tc_commit(&s_full[q]);
      if (last_use) nvb::tc_commit(&k_free[i % KS]);
    };
    auto issue_pv = [&](int q, int i, bool first, bool last_use) {
      const uint64_t vd = v_desc + (uint32_t)(i % VS) * (C::KTILE >> 4);
      const uint32_t d = tmem + C::O_COL + (uint32_t)q * HD, pa = tmem + (uint32_t)q * BN;
      tc_mma_ts(d, pa, vd, IDESC_PV, first ? 0u : 1u);
#pragma unroll
      for (int kk = 1; kk < BN / 16; ++kk) tc_mma_ts(d, pa + kk * 8, vd + kk * (2048 / 16), IDESC_PV, 1u);
      nvb::tc_commit(&o_done[q]);
      if (last_use) nvb::tc_commit(&v_free[i % VS]);
    };
    bool ok = true;
    for (int q = 0; ok && q < (steps1 > 0 ? 2 : steps0); ++q) {  // scores of both tiles' first steps
      const int i = twice ? q : 0;
      ok = wait(&k_full[i % KS], i / KS);
      if (!ok) break;
      nvb::tc_fence_after();
      if (tc_elect()) issue_s(q, i, twice || q == 1);
      __syncwarp();
    }
    for (int j = 0; ok && j < steps0; ++j)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (!ok || (q == 1 && j >= steps1)) break;
        const int i = j * stride + (twice ? q : 0);
        const bool more = j + 1 < (q == 0 ? steps0 : steps1);
        // the tiles are usually there; what the issue waits for is P
        ok = wait(i == nt - 1 && clear ? v_clear : &v_full[i % VS], i == nt - 1 && clear ? 0 : i / VS);
        if (ok && more) ok = wait(&k_full[(i + stride) % KS], (i + stride) / KS);
        if (ok) ok = wait(&p_full[q], j);
        if (!ok) break;
        nvb::tc_fence_after();
        if (tc_elect()) {
          issue_pv(q, i, j == 0, twice || q == 1);
          // the next scores overwrite P: the tensor pipe runs MMAs in the order of issue
          if (more) issue_s(q, i + stride, twice || q == 1);
        }
        __syncwarp();
      }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- V rows behind the prefix
    // They may hold anything: their weight is 0, and 0 * NaN must not reach the sum.
    if (clear) {
      const int i = nt - 1, valid = kend - (t0 + i) * BN;
      if (__all_sync(0xffffffffu, tc_wait(&v_full[i % VS], (uint32_t)((i / VS) & 1), a.err, &abort_flag))) {
        uint8_t* vt = vring + (size_t)(i % VS) * C::KTILE;
        for (int x = lane + valid * (HD / 8); x < BN * (HD / 8); x += 32) {
          const int vr = x / (HD / 8), c = x % (HD / 8);
          *reinterpret_cast<uint4*>(vt + (c >> 3) * C::KBOX + nvb::swz128(vr, c & 7)) = make_uint4(0, 0, 0, 0);
        }
        nvb::fence_proxy_async();
        __syncwarp();
        if (lane == 0) nvb::mbar_arrive(v_clear);
      }
    }
  }
  } else {
    // ---------------------------------------------------------------- softmax and output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int steps = tile == 0 ? steps0 : steps1;
    const bool have = rr < row0 + rows;
    const int t = a.split(rr).x, h = kvh * G + a.split(rr).y;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_col = lanes + (uint32_t)tile * BN, o_col = lanes + C::O_COL + (uint32_t)tile * HD;
    const float sl2 = a.scale * kLog2e;
    const int win = a.window > 0 ? a.window : 0x40000000;
    const bool linear = a.softcap <= 0.f && sl2 > 0.f;  // then the maximum may be taken before the scale
    const float mul = linear ? sl2 : 1.f;
    const bool idle = !have || t >= a.T;  // nothing is written for the row: no need to mask it
    // O and l scaled by f: at the start of a step the product of the step before is done (its scores came after it)
    auto rescale_o = [&](float f) {
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        tc_ld32(o_col + c, o);
        nvb::tmem_ld_wait();
        nvb::reg_fence<32>(o);
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
        tc_st32(o_col + c, o);
      }
    };
    float m_used = -INFINITY, l = 0.f;
    const uint64_t mul2 = pack2(mul, mul);
    bool ok = true;
    for (int j = 0; j < steps; ++j) {
      if (!__all_sync(0xffffffffu, tc_wait(&s_full[tile], (uint32_t)(j & 1), a.err, &abort_flag))) {
        ok = false;
        break;
      }
      nvb::tc_fence_after();
      const int key0 = (t0 + j * stride + (twice ? tile : 0)) * BN;
      // columns (lo, hi] are seen; a key tile that every row of this warp sees whole skips the masks
      const int hi = min(kend - 1, pos) - key0, lo = pos - win - key0;
      const bool whole = __all_sync(0xffffffffu, idle || (hi >= BN - 1 && lo < 0));
      uint64_t rs0 = 0, rs1 = 0;
      // 32 columns at a time in a loop, not unrolled: instructions arrive at about one a clock the first time, and the
      // whole tile unrolled made a CTA's first step take 14000 clocks where the others take 3400.
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        uint32_t u[32];
        tc_ld32(s_col + c, u);
        nvb::tmem_ld_wait();
        nvb::reg_fence<32>(u);
        auto val = [&](int e) { return __uint_as_float(u[e]); };
        if (!linear) {
          if (a.softcap > 0.f) {
#pragma unroll
            for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(sp_cap(val(e) * a.scale, a.softcap) * kLog2e);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(val(e) * sl2);
          }
        }
        if (!whole) {
#pragma unroll
          for (int e = 0; e < 32; ++e) u[e] = c + e <= hi && c + e > lo ? u[e] : 0xff800000u;
        }
        // The weights are taken against the maximum in use before these columns' is known: it holds for most of them, and
        // theirs is found on the way.  Only where there is none yet it is taken first.
        if (!__all_sync(0xffffffffu, m_used > -INFINITY)) {
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; e += 2) m4[(e >> 1) & 3] = fmaxf(fmaxf(val(e), val(e + 1)), m4[(e >> 1) & 3]);
          const float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * mul;
          if (m_used == -INFINITY && mt > -INFINITY) m_used = mt;  // O and the weights before are still zero
        }
        const float mneg = m_used == -INFINITY ? 0.f : -m_used;  // without keys every score is -inf, every weight 0
        const uint64_t neg2 = pack2(mneg, mneg);
        uint32_t w[16];
        uint64_t sum0 = 0, sum1 = 0;
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint64_t v = fma2(pack2(val(e), val(e + 1)), mul2, neg2);
          const int pair = (e / 2) % 8;
          float p0, p1;
          unpack2(v, p0, p1);
          top4[pair & 3] = fmaxf(fmaxf(p0, p1), top4[pair & 3]);
          if (pair == 1 || pair == 4 || pair == 6) {
            exp2_poly2(v, p0, p1);
          } else {
            p0 = exp2f(p0);
            p1 = exp2f(p1);
          }
          if (pair & 1) sum1 = add2(sum1, pack2(p0, p1));
          else sum0 = add2(sum0, pack2(p0, p1));
          w[e / 2] = nvb::pack_bf16x2(p0, p1);
        }
        const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        if (__any_sync(0xffffffffu, top > 8.f)) {
          // The maximum in use moves; O, l, the weights of the columns before and these ones follow.  By a whole power of
          // two, so that weights which have been rounded to bf16 are not rounded again.
          const float up = top > 8.f ? ceilf(top) : 0.f;
          const float f = up > 126.f ? 0.f : __int_as_float((127 - (int)up) << 23);
          m_used += up;
          if (j > 0) rescale_o(f);
          l *= f;
          rs0 = fma2(rs0, pack2(f, f), 0), rs1 = fma2(rs1, pack2(f, f), 0);
          tc_st_wait();
#pragma unroll 1
          for (int d = 0; d < c; d += 32) {
            uint32_t q[16];
            nvb::tmem_ld_32x32b_x16(s_col + d / 2, q);
            nvb::tmem_ld_wait();
            nvb::reg_fence<16>(q);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              q[e] = nvb::pack_bf16x2(__uint_as_float(q[e] << 16) * f, __uint_as_float(q[e] & 0xffff0000u) * f);
            tc_st16(s_col + d / 2, q);
          }
          const float now = m_used == -INFINITY ? 0.f : -m_used;
          sum0 = sum1 = 0;
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float p0 = exp2f(fmaf(val(e), mul, now)), p1 = exp2f(fmaf(val(e + 1), mul, now));
            sum0 = add2(sum0, pack2(p0, p1));
            w[e / 2] = nvb::pack_bf16x2(p0, p1);
          }
        }
        rs0 = add2(rs0, sum0), rs1 = add2(rs1, sum1);
        tc_st16(s_col + c / 2, w);  // over scores that have been read
      }
      float r0, r1;
      unpack2(add2(rs0, rs1), r0, r1);
      l += r0 + r1;
      tc_st_wait();
      nvb::tc_fence_before();
      __syncwarp();
      if (lane == 0) nvb::mbar_arrive(&p_full[tile]);
    }
    // the part: O / l and the log2-sum-exp
    int okw = ok ? 1 : 0;
    if (ok && steps > 0 && lane == 0) okw = tc_wait(&o_done[tile], (uint32_t)((steps - 1) & 1), a.err, &abort_flag) ? 1 : 0;
    okw = __shfl_sync(0xffffffffu, okw, 0);
    nvb::tc_fence_after();
    asm volatile("bar.sync 2, 256;" ::: "memory");  // both tiles' products are done: the rings are free
    if (okw && *reinterpret_cast<volatile int*>(&abort_flag) == 0 && have) {
      const int NS = pl.slots(), part = 2 * split + (twice ? tile : 0);
      const long slot = ((long)t * a.nq + h) * NS + part;
      pl.part_lse[slot] = l > 0.f ? m_used + log2f(l) : -INFINITY;
      if (!twice) pl.part_lse[slot + 1] = -INFINITY;
    }
    if (okw && *reinterpret_cast<volatile int*>(&abort_flag) == 0 && steps > 0) {
      // Each thread lays its row of O into shared memory (rows 16 bytes more than their length apart: no bank conflicts)
      // and copies it out as a whole: stores of 64 bytes a row took 9000 clocks for 256 rows, these a third of it.
      constexpr int PITCH = HD * 4 + 16;
      static_assert(256 * PITCH <= (KS + VS) * C::KTILE, "rows of O in the rings");
      const float inv = l > 0.f ? 1.f / l : 0.f;
      uint8_t* st = kring + (tile * 128 + r) * PITCH;
#pragma unroll 1
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        tc_ld32(o_col + c, o);
        nvb::tmem_ld_wait();
        nvb::reg_fence<32>(o);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<float4*>(st + c * 4 + k * 16) =
              make_float4(__uint_as_float(o[4 * k]) * inv, __uint_as_float(o[4 * k + 1]) * inv,
                          __uint_as_float(o[4 * k + 2]) * inv, __uint_as_float(o[4 * k + 3]) * inv);
      }
      nvb::fence_proxy_async();
      if (have) {
        const float* dst = pl.part_o + (((long)t * a.nq + h) * pl.slots() + 2 * split + (twice ? tile : 0)) * HD;
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(nvb::smem_u32(st)),
                     "r"(HD * 4)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory");
      }
    }
  }
  nvb::tc_fence_before();
  __syncthreads();
  nvb::tc_fence_after();
  if (warp == 1) nvb::tmem_dealloc(tmem, 512);
}

template <int HD>
void launch_tc(const SpArgs& a, const SpPlan& pl, const void* kc, const void* vc, cudaStream_t stream) {
  const uint64_t rows = (uint64_t)a.num_blocks * a.nkv * a.block_size;
  const CUtensorMap km = nvb::make_tmap_2d_bf16(kc, rows, HD, HD, SpTc<HD>::BN);
  const CUtensorMap vm = nvb::make_tmap_2d_bf16(vc, rows, HD, HD, SpTc<HD>::BN);
  auto kern = sp_tc_kernel<HD>;
  constexpr size_t sm = SpTc<HD>::smem();
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sm));
  C10_CUDA_CHECK(nvb::launch(kern, dim3((unsigned)(pl.n_pre * a.nkv * pl.pre_row_tiles)), dim3(384), sm, stream, km, vm, a, pl));
}
