// Backward of the attention: dQ, dK, dV and the gradient of the bucketed relative position
// bias, for every form of the forward (full, window and sinks, ALiBi, bias table, dropout).
//
// With P_ij = exp(t_ij - lse_i) recomputed from the scores and the saved lse, m_ij the
// dropout multiplier and delta_i = sum_d dO_id O_id (which equals sum_j P_ij m_ij dO_i.v_j):
//   dV_j = sum_i m_ij P_ij dO_i
//   dS_ij = P_ij (m_ij dO_i . v_j - delta_i)
//   dQ_i = scale sum_j dS_ij k_j,   dK_j = scale sum_i dS_ij q_i
//   dTable[b, h] = sum of dS_ij over the pairs with bucket(j - i) = b
//
// Two passes, so that every sum has a fixed order and no atomics: dq_kernel keeps 32 queries
// per wave and walks the key tiles (3 products a tile: scores, dP, dQ), dkv_kernel keeps 32
// keys per wave and walks the query tiles of each query head that shares the key head (4
// products).  That is 7 products for the formulas' 5.  Both form the scores so that the
// wave's own rows are the columns of the product (attn_tile.h): P and dS then are B operands
// as they stand.  P and dS enter the products as bf16 (sums in fp32), as P does in the
// forward: a value's rounding is 2^-8 relative, of random sign, and the sums average over it.
//
// What bounds it: matrix and vector instructions together.  Counters, all SIMDs, 8 x 4,550
// tokens, 12 heads, ALiBi: dq_kernel matrix units busy 38 %, vector issue 44 %; dkv_kernel 40
// and 39 %, LDS reads 29 % without a bank conflict; 2 x 4,550 with buckets 30 and 45, 34 and
// 33 % at 1.45 of 2 waves per SIMD (864 workgroups on 512 places).
// Measured (dq_kernel, dkv_kernel; 12 heads; rates of the 3 and 4 products): 8 x 4,550 tokens
// without options 745, 1,060 us (1,024, 960 TFLOP/s); buckets 2 x 4,550 284, 326 us (672, 780),
// 16 x 512 59, 53 us; window of 1,024 + 1,024 over 1 x 9,000 120, 157 us; ALiBi 8 x 4,550 360,
// 444 us.
#include <algorithm>
#include <type_traits>

#include "attn_tile.h"

namespace g5moe {
namespace attn {
namespace {

constexpr int kPairQ = 2 * kTileBytes;         // dq_kernel: K tile, V tile
constexpr int kVecBytes = 1024;                // dkv_kernel: -lse, -delta, row keys of a tile
constexpr int kPairKV = 2 * kTileBytes + kVecBytes;

// A wave adds up dS by distance in a table of its own in LDS, so the order of its sums is
// fixed.  A 32 x 32 block of dS is first summed along its diagonals: the block goes through
// LDS (row: query, kDiagPitch floats apart), and lane d of either half wave reads, for its 16
// queries q, key (q + d) % 32.  Those with q + d < 32 lie on diagonal d, the others on d - 32,
// so each element is read once; the reads of a step are consecutive, the pitch keeps the
// 8-byte writes and the reads off each other's banks.  (One LDS float atomic per element
// instead takes two cycles a lane: 16 x 512 tokens, 12 heads, 193 us for dq_kernel.)
constexpr int kGradTables = 4;
constexpr int kDiagPitch = 34;
constexpr int kDiagFloats = kCols * kDiagPitch;   // per wave

// dq_kernel's waves per SIMD: three without a position bias, whose code fits 160 registers (12
// heads, two against three: 8 x 4,550 tokens 818, 742 us; 2 x 4,550 230, 227; window of 256 + 256
// over 8 x 2,048 72, 64).  ALiBi would spill three registers or subtract delta again, and its
// launches of less than two rounds lose (8 x 4,550 366, 355; 2 x 4,550 105, 122; 4 x 1,100 35, 39);
// the tables of the bias gradient leave LDS for two workgroups per CU.
constexpr int dq_waves(int pos) { return pos == kPosNone ? 3 : 2; }

template <int POS, bool DROP, bool DBIAS, bool WIDE, int KS>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(dq_waves(POS), dq_waves(POS))))
void dq_kernel(LocalArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  using S = Split<KS>;
  constexpr int kStageQ = KS * kPairQ;
  char* const ring = smem;
  float* const tab = reinterpret_cast<float*>(smem + S::kStages * kStageQ);
  const int n_tab = POS == kPosTable ? bias_entries(a.far) : 0;
  float* const gtab = tab + n_tab;
  float* const diag = gtab + (DBIAS ? kGradTables * n_tab + (n_tab & 1) : 0);  // 8-byte aligned

  int slot, hq;
  if (!block_of(blockIdx.x, a.qb.count, a.n_heads, slot, hq)) return;
  if (POS == kPosAlibi && a.kmax != nullptr && a.n_heads <= 64)
    hq = by_slope(a.slopes, a.n_heads, hq);
  zero_tail(a, a.dq, a.dq_tok, hq * a.dq_head, slot, a.qb.count);
  int z, s0, L, q0;
  if (!find_block(a, a.qb, slot, z, s0, L, q0)) {
    if constexpr (DBIAS) {  // the sums by distance of no query
      const int E = 2 * a.far + 1;
      float* out = a.part + (int64_t(hq) * a.qb.count + slot) * E;
      for (int x = threadIdx.x; x < E; x += 256) out[x] = 0.0f;
    }
    return;
  }
  const int hk = hq / a.group;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int tg = S::tile(wave);
  const int wq = q0 + S::own(wave) * kCols;
  const int wq_hi = min(wq + kCols, L) - 1;
  const int iq = wq + col;
  const bool own = iq < L;
  const int wl = min(a.wl, L), wr = min(a.wr, L), ns = min(a.ns, L);
  const float sc = a.sc;
  const float sl = POS == kPosAlibi ? a.slopes[hq] * kLog2e : 0.0f;

  bf16x8 qf[4], dof[4];
  OwnRows qr, dor, orw, low = {};
  float lse;
  {
    const int64_t t = s0 + min(iq, L - 1);
    qr.request(a.q + t * a.q_tok + hq * a.q_head, half);
    lse = a.lse[int64_t(hq) * a.total + t];
    dor.request(a.dout + t * a.do_tok + hq * a.do_head, half);
    orw.request(a.o + t * a.o_tok + hq * a.o_head, half);
    if (a.o_low != nullptr) low.request(a.o_low + (t * a.n_heads + hq) * kHeadDim, half);
  }
  KeyTiles kt;
  TilePair<WIDE> tiles;
  tiles.init(ring, wave, lane, L, a.k_tok * 2, a.v_tok * 2);
  FragReader fr;
  fr.init(lane);
  const char* const kbase =
      reinterpret_cast<const char*>(a.k + int64_t(s0) * a.k_tok + hk * a.k_head);
  const char* const vbase =
      reinterpret_cast<const char*>(a.v + int64_t(s0) * a.v_tok + hk * a.v_head);
  // past the last tile it goes out again, into a buffer that no later tile reads
  int n_is = 0;
  auto issue = [&](uint32_t boff) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < KS; ++g) {
      tiles.issue(kbase, vbase, __builtin_amdgcn_readfirstlane(n_is), boff + g * kPairQ);
      n_is = n_is < kt.w_hi ? kt.next(n_is) : n_is;
    }
  };
  auto begin = [&](int reach) __attribute__((always_inline)) {
    kt.init(q0, min(q0 + S::kOwn, L) - 1, L, min(wl, reach), min(wr, reach),
            q0 - (ns - 1) > reach ? 0 : ns);
    n_is = kt.first();
#pragma unroll
    for (int st = 0; st < S::kStages; ++st) issue(uint32_t(st) * kStageQ);
  };
  if constexpr (POS != kPosAlibi) begin(L);
  qr.take(qf, own, 0u);
  // a row past the end has probabilities of 0; of an empty row every term is -inf, whatever
  // is subtracted
  float nl = !own ? -kInf : lse == -kInf ? 0.0f : -lse * kLog2e;
  asm volatile("" : "+v"(nl));
  if constexpr (POS == kPosAlibi) {
    // With the key norms, keys farther than `reach` from every query of the workgroup are left
    // out: P_ij <= 2^(|q||k| sc - sl |i - j| - lse_i log2(e)) < 2^-40 there.
    int reach = L;
    if (a.kmax != nullptr) {
      float v[2] = {norm_max(qf), nl};
      __shared__ float red[2][4];
      block_max(v, red, wave, lane);
      const float bound = __builtin_fabsf(sc) * v[0] * key_norm(a, hk, s0, L, red, wave, lane);
      reach = alibi_reach(bound + v[1], sl, L);
      if (tid == 0)
        a.qmax[int64_t(hq) * a.qb.count + slot] = float2{v[0], v[1]};
    }
    begin(reach);
  }
  dor.take(dof, own, 0u);
  float delta = 0.0f;
  {
    // The rounding of o alone would leave an error in delta that enters dS with the weight P:
    // of a row with few keys of weight it would be a large part of the error (ALiBi: dq and dk
    // 2.6e-3 without o_low, 2.4e-3 with).
    bf16x8 of[4], lf[4];
    orw.take(of, own, 0u);
    low.take(lf, own, 0u);
#pragma unroll
    for (int kc = 0; kc < 4; ++kc)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        delta = __builtin_fmaf(float(dof[kc][e]), float(of[kc][e]) + float(lf[kc][e]), delta);
    delta += __shfl_xor(delta, 32, 64);
  }
  uint32_t rkey = 0, thr = 0;
  float up = 0.0f;
  if constexpr (DROP) {
    rkey = dropout_row_key(uint32_t(s0 + iq) * uint32_t(a.n_heads) + uint32_t(hq),
                           a.drop.seed_lo, a.drop.seed_hi);
    thr = min(a.drop.thr, 65535u) << 16;  // p = 1: the scale is 0
    up = a.drop.scale;
  }
  if constexpr (POS == kPosTable) stage_bias(a, hq, tab);
  if constexpr (DBIAS)
    for (int x = tid; x < kGradTables * n_tab; x += 256) gtab[x] = 0.0f;
  if constexpr (POS == kPosTable) __syncthreads();
  const float far_l = POS == kPosTable ? tab[0] : 0.0f;
  const float far_r = POS == kPosTable ? tab[n_tab - 1] : 0.0f;
  BiasChunk bc;
  if constexpr (POS == kPosAlibi) bc.init(sl, sc, lane);

  // -delta to start the product dP from, which saves its subtraction; with dropout it follows
  // the multiplier
  f32x16 dp0 = {};
  if constexpr (!DROP)
#pragma unroll
    for (int r = 0; r < 16; ++r) dp0[r] = -delta;

  f32x16 dq[2] = {f32x16{}, f32x16{}};
  // DBIAS, per query: sums of dS and P in the far tiles (distances <= -far and >= far), and of
  // dS in the others
  float sum_l = 0.0f, sum_r = 0.0f, p_l = 0.0f, p_r = 0.0f, sum_near = 0.0f;

  // dS of 32 keys: half b of tile n, scores s and dP dp; c: the tile's constant bias.
  auto grad = [&](auto mask_c, auto look_c, int n, int b, const f32x16& s, const f32x16& dp,
                  float c, bool left, uint32_t (&pk)[8]) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_c)::value, LOOK = decltype(look_c)::value;
    const int j0 = n * kRows + 32 * b + 4 * half;
    const int lo = iq - wl - j0;
    const uint32_t span = uint32_t(min(iq + wr, L - 1) - (iq - wl));
    const int sink = ns - j0;
    const float di = float(iq - j0);
    const float* tb = tab + (j0 - iq + a.far + kBiasPad);
    float* const dg = diag + wave * kDiagFloats;
    const uint32_t jp = uint32_t(j0) >> 1;
    const float sub = nl + c;
    float sum = 0.0f, p_sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      uint32_t bits = 0;
      if constexpr (DROP) bits = dropout_pair_bits(rkey, jp + uint32_t(8 * (r >> 2) + (r & 3)) / 2);
      float ds[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int kr = 8 * (r >> 2) + (r & 3) + e;
        const float x = s[r + e];
        float t;
        if constexpr (LOOK && POS == kPosTable)
          t = __builtin_fmaf(x, sc, tb[kr]) + nl;
        else if constexpr (LOOK && POS == kPosAlibi)
          t = __builtin_fmaf(-sl, __builtin_fabsf(di - float(kr)), x * sc) + nl;
        else
          t = __builtin_fmaf(x, sc, sub);
        if constexpr (MASK) t = (uint32_t(kr - lo) <= span || kr < sink) ? t : -kInf;
        const float p = __builtin_amdgcn_exp2f(t);
        float d = dp[r + e];
        if constexpr (DROP) {
          const bool keep =
              e == 0 ? uint16_t(bits) >= uint16_t(thr >> 16) : bits >= thr;
          const float mult = keep ? up : 0.0f;
          d = __builtin_fmaf(d, mult, -delta);
        }
        ds[e] = p * d;
        if constexpr (DBIAS) sum += ds[e];
        if constexpr (DBIAS && !LOOK) p_sum += p;
      }
      if constexpr (DBIAS && LOOK)
        *reinterpret_cast<float2*>(dg + col * kDiagPitch + 8 * (r >> 2) + 4 * half + (r & 3)) =
            float2{ds[0], ds[1]};
      pk[r >> 1] = pack_bf16x2(ds[0], ds[1]);
    }
    if constexpr (DBIAS && LOOK) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      float all = 0.0f, on = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = dg[(16 * half + i) * kDiagPitch + ((16 * half + i + col) & 31)];
        all += x;
        on = __builtin_fmaf(x, 16 * half + i + col < 32 ? 1.0f : 0.0f, on);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      all += __shfl_xor(all, 32, 64);
      on += __shfl_xor(on, 32, 64);
      // lanes 0 .. 31: diagonal col; lanes 32 .. 63: col - 32
      gtab[wave * n_tab + (n * kRows + 32 * b - wq + a.far + kBiasPad) + col - 32 * half] +=
          half == 0 ? on : all - on;
    }
    if constexpr (DBIAS && LOOK) sum_near += sum;
    if constexpr (DBIAS && !LOOK) {
      sum_l += left ? sum : 0.0f;
      sum_r += left ? 0.0f : sum;
      p_l += left ? p_sum : 0.0f;
      p_r += left ? 0.0f : p_sum;
    }
  };

  int n = kt.first();
  if (tg == 1) n = kt.next(n);
  uint32_t boff = 0;
  gemm::wait_vmcnt<(S::kStages - 1) * 4 * KS>();
  __syncthreads();
  for (int left = kt.count(); left > 0; left -= KS) {
    const int j0 = n * kRows, j1 = j0 + kRows - 1;
    const bool some =
        left > tg && wq < L && ((j0 <= wq_hi + wr && j1 >= wq - wl) || j0 < ns);
    if (some) {
      const f32x16 zero16 = {};
      const char* const K = ring + boff + tg * kPairQ;
      const char* const V = K + kTileBytes;
      const bool all = j1 < L && ((j0 >= wq_hi - wl && j1 <= wq + wr) || j1 < ns);
      using T_ = std::true_type;
      using F_ = std::false_type;
      float c = 0.0f;
      bool look = false, far_left = false, before = false;
      if constexpr (POS == kPosTable) {
        far_left = j1 - wq <= -a.far;
        look = !far_left && j0 - wq_hi < a.far;
        c = far_left ? far_l : far_r;
      }
      if constexpr (POS == kPosAlibi) {
        before = j1 <= wq;
        look = !(bc.ok && (before || j0 >= wq_hi));
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x16 s, dp;
#pragma unroll
        for (int kc = 0; kc < 4; ++kc)
          s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.row(K, b, kc), qf[kc],
                                                      kc == 0 ? zero16 : s, 0, 0, 0);
#pragma unroll
        for (int kc = 0; kc < 4; ++kc)
          dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.row(V, b, kc), dof[kc],
                                                       kc == 0 ? dp0 : dp, 0, 0, 0);
        uint32_t pk[8];
        if constexpr (POS == kPosAlibi)
          if (!look) s = bc.add_half(s, b, float(iq - j0), before);
        if (POS != kPosNone && look) {
          if (all)
            grad(F_{}, T_{}, n, b, s, dp, 0.0f, false, pk);
          else
            grad(T_{}, T_{}, n, b, s, dp, 0.0f, false, pk);
        } else {
          if (all)
            grad(F_{}, F_{}, n, b, s, dp, c, far_left, pk);
          else
            grad(T_{}, F_{}, n, b, s, dp, c, far_left, pk);
        }
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const bf16x8 df = chunk(pk, cc);
#pragma unroll
          for (int mb = 0; mb < 2; ++mb)
            dq[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.trans(K, 2 * b + cc, mb), df,
                                                             dq[mb], 0, 0, 0);
        }
      }
    }
    // the next stage landed, and every wave has read all of this one
    gemm::wait_vmcnt<(S::kStages - 2) * 4 * KS>();
    __syncthreads();
    issue(boff);
    boff = boff + kStageQ == S::kStages * kStageQ ? 0 : boff + kStageQ;
#pragma unroll
    for (int g = 0; g < KS; ++g) n = kt.next(n);
  }
  // refills past the last tile may still be landing in this workgroup's LDS
  gemm::wait_vmcnt<0>();

  if (own && half == 0 && tg == 0) {  // for dkv_kernel
    const int64_t at = int64_t(hq) * a.total + s0 + iq;
    a.nl[at] = nl;
    a.delta[at] = -delta;
    if constexpr (DROP) a.rowkey[at] = rkey;
  }
  bool holds = true;
  if constexpr (KS == 2) {
    float v[32];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      v[r] = dq[0][r];
      v[16 + r] = dq[1][r];
    }
    holds = join_waves(v, ring, wave, lane);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dq[0][r] = v[r];
      dq[1][r] = v[16 + r];
    }
  }
  if (own && holds) {
    uint16_t* op = a.dq + int64_t(s0 + iq) * a.dq_tok + hq * a.dq_head + 4 * half;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint2 w;
        w.x = pack_bf16x2(dq[mb][4 * q] * a.scale, dq[mb][4 * q + 1] * a.scale);
        w.y = pack_bf16x2(dq[mb][4 * q + 2] * a.scale, dq[mb][4 * q + 3] * a.scale);
        *reinterpret_cast<uint2*>(op + 32 * mb + 8 * q) = w;
      }
  }

  if constexpr (DBIAS) {
    // the workgroup's sums by distance, clamped to +-far, in a fixed order: the tables in
    // order, then what lies past far, then the plain tiles' sums
    // A row of dS sums to zero; what it sums to here is the error that the rounding of the
    // forward's probabilities leaves in delta.  It enters every term with the weight P, so the
    // two end buckets, which hold most of P in long sequences while their own terms nearly
    // cancel, are corrected by it (relative error of the table's gradient up to 3.4e-3 without,
    // 1.1e-3 to 2.1e-3 with, for 7 % of dq_kernel's time at 2 x 4,550 tokens); the others hold a
    // share of P that is too small to matter.
    __shared__ float ends[2][4];
    {
      const float row = sum_l + sum_r + sum_near;
      const float err = row + __shfl_xor(row, 32, 64);
      sum_l = __builtin_fmaf(-err, p_l, sum_l);
      sum_r = __builtin_fmaf(-err, p_r, sum_r);
    }
    sum_l = butterfly_sum64(sum_l);
    sum_r = butterfly_sum64(sum_r);
    if (lane == 0) {
      ends[0][wave] = sum_l;
      ends[1][wave] = sum_r;
    }
    __syncthreads();
    auto column = [&](int x) {
      float v = 0.0f;
#pragma unroll
      for (int t = 0; t < kGradTables; ++t) v += gtab[t * n_tab + x];
      return v;
    };
    const int E = 2 * a.far + 1;
    float* out = a.part + (int64_t(hq) * a.qb.count + slot) * E;
    for (int x = tid; x < E; x += 256)
      if (x != 0 && x != E - 1) out[x] = column(kBiasPad + x);
    if (wave < 2) {
      // entries 0 .. kBiasPad (left) or the last kBiasPad + 1 (right)
      const int from = wave == 0 ? 0 : kBiasPad + E - 1;
      float v = column(from + lane);
      if (lane < kBiasPad + 1 - 64) v += column(from + 64 + lane);
      v = butterfly_sum64(v);
      v += ends[wave][0] + ends[wave][1] + (ends[wave][2] + ends[wave][3]);
      if (lane == 0) out[wave == 0 ? 0 : E - 1] = v;
    }
  }
}

// The gradient of one head's column of the bias table, by one workgroup: the sums by distance
// of dq_kernel's workgroups added up in order (those of unused numbers wrote zeros), then those
// of each bucket.  E distances, a thread per distance and (up to 256) stretch of the workgroups.
__device__ __forceinline__ void bias_grad(const LocalArgs& a, int h, float* rel) {
  const int E = 2 * a.far + 1;
  const int64_t n = a.qb.count;
  const float* const p = a.part + int64_t(h) * n * E;
  for (int x = threadIdx.x; x < E; x += 256) {
    float v[8] = {};
    int64_t i = 0;
    for (; i + 8 <= n; i += 8)
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] += p[(i + u) * E + x];
    for (; i < n; ++i) v[0] += p[i * E + x];
    rel[x] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  }
  int* const bucket = reinterpret_cast<int*>(rel + E);
  for (int x = threadIdx.x; x < E; x += 256)
    bucket[x] = min(max(a.bucket_of[x], 0), a.n_buckets - 1);
  __syncthreads();
  for (int b = threadIdx.x; b < a.n_buckets; b += 256) {
    float sum = 0.0f;
    for (int x = 0; x < E; ++x) sum += bucket[x] == b ? rel[x] : 0.0f;
    const int64_t at = int64_t(b) * a.n_heads + h;
    if (a.bias_bf16)
      static_cast<uint16_t*>(a.dbias)[at] = f32_to_bf16_bits(sum);
    else
      static_cast<float*>(a.dbias)[at] = sum;
  }
}

// dkv_kernel's workgroups per head.
__host__ __device__ __forceinline__ int kv_units(const LocalArgs& a) {
  return a.n_seqs * a.sink_blocks * a.sink_splits + a.kb.count * a.splits;
}

// 32 keys per wave against the tiles of queries (Q, dO and their -lse, -delta, row keys).  The
// tiles of a key block (of each query head that shares the key head) may be split over several
// workgroups, `splits` of them or `sink_splits` for the blocks that hold sinks, which every
// query sees: each writes its sums in fp32 and kv_join_kernel adds them up in order.
template <int POS, bool DROP, bool WIDE, int KS>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2, 2)))
void dkv_kernel(LocalArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  using S = Split<KS>;
  constexpr int kStageKV = KS * kPairKV;
  char* const ring = smem;
  float* const tab = reinterpret_cast<float*>(smem + S::kStages * kStageKV);

  // the first workgroups reduce the bias gradient, behind which the others' work hides
  uint32_t id = blockIdx.x;
  if constexpr (POS == kPosTable) {
    if (a.dbias != nullptr) {
      if (id < uint32_t(a.n_heads)) {
        bias_grad(a, int(id), reinterpret_cast<float*>(smem));
        return;
      }
      id -= uint32_t(a.n_heads);
    }
  }
  int unit, hk;
  if (!block_of(id, kv_units(a), a.n_heads / a.group, unit, hk)) return;
  if (POS == kPosAlibi && a.qmax != nullptr && a.group == 1 && a.n_heads <= 64)
    hk = by_slope(a.slopes, a.n_heads, hk);
  zero_tail(a, a.dk, a.dk_tok, hk * a.dk_head, unit, kv_units(a));
  zero_tail(a, a.dv, a.dv_tok, hk * a.dv_head, unit, kv_units(a));
  // the sinks' blocks first: theirs is the longest work
  const int n_sink = a.n_seqs * a.sink_blocks * a.sink_splits;
  const bool sink_block = unit < n_sink;
  const int splits = sink_block ? a.sink_splits : a.splits;
  const int block = (sink_block ? unit : unit - n_sink) / splits;
  const int split = (sink_block ? unit : unit - n_sink) % splits;
  int z, s0, L, k0;
  if (sink_block) {
    z = block / a.sink_blocks;
    sequence(a, z, s0, L);
    k0 = block % a.sink_blocks * S::kOwn;
    if (k0 >= L) return;
  } else if (!find_block(a, a.kb, block, z, s0, L, k0) || k0 < a.sink_blocks * S::kOwn) {
    return;
  }
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int tg = S::tile(wave);
  const int wk = k0 + S::own(wave) * kCols;               // the wave's keys: wk .. wk_hi
  const int wk_hi = min(wk + kCols, L) - 1;
  const int jk = wk + col;
  const bool own = jk < L;
  const int wl = min(a.wl, L), wr = min(a.wr, L), ns = min(a.ns, L);
  const float sc = a.sc;

  bf16x8 kf[4], vf[4];
  OwnRows kr, vr;
  kr.request(a.k + int64_t(s0 + min(jk, L - 1)) * a.k_tok + hk * a.k_head, half);
  vr.request(a.v + int64_t(s0 + min(jk, L - 1)) * a.v_tok + hk * a.v_head, half);
  uint32_t thr = 0, golden_c = 0;
  const uint32_t low = (lane & 1) ? 0 : 16;  // an even key takes the low half of a hash
  float up = 0.0f;
  if constexpr (DROP) {
    thr = min(a.drop.thr, 65535u) << 16;
    golden_c = (uint32_t(jk) >> 1) * 0x9e3779b9u;
    up = a.drop.scale;
  }
  if constexpr (POS == kPosAlibi) kr.take(kf, own, 0u);

  // query tiles that see one of the workgroup's keys; with ALiBi and norms not those farther
  // than `reach` from all of them, by the same bound
  int reach = L;
  if (POS == kPosAlibi && a.qmax != nullptr) {
    __shared__ float red[2][4];
    float kn[1] = {norm_max(kf)};
    block_max(kn, red, wave, lane);
    reach = 0;
    for (int g = 0; g < a.group; ++g) {
      const int h = hk * a.group + g;
      const float2* p = a.qmax + int64_t(h) * a.qb.count + a.qb.first(z, s0);
      float top[1] = {-kInf};
      for (int i = tid; i << a.qb.shift < L; i += 256)
        top[0] = __builtin_fmaxf(top[0],
                                 __builtin_fmaf(__builtin_fabsf(sc) * kn[0], p[i].x, p[i].y));
      block_max(top, red, wave, lane);
      reach = max(reach, alibi_reach(top[0], a.slopes[h] * kLog2e, L));
    }
  }
  const int k_hi = min(k0 + S::kOwn, L) - 1;
  const int t_lo = k0 < ns && reach == L ? 0
                   : max(k0 - min(k0 < ns ? L : wr, reach), 0) / kRows;
  const int t_hi = min(k_hi + min(k0 < ns ? L : wl, reach), L - 1) / kRows;
  // this workgroup's share of (head, tile) in order: (h_a, n_a) .. (h_b, n_b)
  const int n_t = t_hi - t_lo + 1;
  const int n_all = n_t * a.group;
  const int f_a = int(int64_t(n_all) * split / splits);
  const int f_b = int(int64_t(n_all) * (split + 1) / splits) - 1;
  const bool work = f_a <= f_b;
  const int h_a = hk * a.group + f_a / n_t, n_a = t_lo + f_a % n_t;
  const int h_b = hk * a.group + f_b / n_t, n_b = t_lo + f_b % n_t;

  TilePair<WIDE> tiles;
  tiles.init(ring, wave, lane, L, a.q_tok * 2, a.do_tok * 2);
  FragReader fr;
  fr.init(lane);
  const uint32_t vec_off[2] = {uint32_t(lane) * 4, uint32_t(min(lane, tiles.lastrow)) * 4};
  const uint32_t vec_lds = gemm::lds_addr(ring) + 2 * kTileBytes + uint32_t(wave) * 256;
  const float* const vsrc = wave == 1 ? a.delta
                            : (DROP && wave == 2) ? reinterpret_cast<const float*>(a.rowkey)
                                                  : a.nl;
  // KS tiles of one head at a time, the last of a head's repeated where there is none left;
  // past the last step it goes out again
  int h_is = h_a, n_is = n_a, n_stop = h_a == h_b ? n_b : t_hi;
  auto issue = [&](uint32_t boff) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < KS; ++g) {
      const int h = __builtin_amdgcn_readfirstlane(h_is);
      const int n = __builtin_amdgcn_readfirstlane(min(n_is + g, n_stop));
      tiles.issue(reinterpret_cast<const char*>(a.q + int64_t(s0) * a.q_tok + h * a.q_head),
                  reinterpret_cast<const char*>(a.dout + int64_t(s0) * a.do_tok + h * a.do_head),
                  n, boff + g * kPairKV);
      gemm::lds_dma4_s(vsrc + int64_t(h) * a.total + s0 + int64_t(n) * kRows,
                       n == tiles.last ? vec_off[1] : vec_off[0], vec_lds + boff + g * kPairKV);
    }
    if (n_is + KS <= n_stop) {
      n_is += KS;
    } else if (h_is < h_b) {
      ++h_is;
      n_is = t_lo;
      n_stop = h_is == h_b ? n_b : t_hi;
    }
  };

  f32x16 dk[2] = {f32x16{}, f32x16{}}, dv[2] = {f32x16{}, f32x16{}};
  float sl = 0.0f, far_l = 0.0f, far_r = 0.0f;
  BiasChunk bc;

  // P (dropped) and dS of 32 queries: half b of tile n, scores s and dP dp.
  auto grad = [&](auto mask_c, auto look_c, int n, int b, const f32x16& s, const f32x16& dp,
                  float c, uint32_t pair, uint32_t (&pkp)[8], uint32_t (&pkd)[8])
      __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_c)::value, LOOK = decltype(look_c)::value;
    const int i0 = n * kRows + 32 * b + 4 * half;
    // tile offsets of the queries that see key jk: lo .. lo + span
    const bool sink = jk < ns;
    const int q_lo = sink ? 0 : max(jk - wr, 0);
    const int q_hi = sink ? L - 1 : min(jk + wl, L - 1);
    const int lo = q_lo - i0;
    const uint32_t span = uint32_t(q_hi - q_lo);
    const float dj = float(jk - i0);
    const float* tb = tab + (jk - i0 - 31 + a.far + kBiasPad);
    const float* vec =
        reinterpret_cast<const float*>(ring + pair + 2 * kTileBytes) + 32 * b + 4 * half;
    uint32_t hb[8];
    if constexpr (DROP) {
      // a pair of lanes being the two columns of one hash, even lanes hash for the first 16
      // queries, odd lanes for the others
      const uint32_t* keys = reinterpret_cast<const uint32_t*>(vec) + 128 + 16 * (lane & 1);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const u32x4 kk = *reinterpret_cast<const u32x4*>(keys + 8 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) hb[4 * q + e] = fmix32(kk[e] + golden_c);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4 nl4 = *reinterpret_cast<const f32x4*>(vec + 8 * q);
      f32x4 dl4;
      if constexpr (DROP) dl4 = *reinterpret_cast<const f32x4*>(vec + 64 + 8 * q);
      float pd[4], ds[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * q + e;
        const int qr = 8 * q + e;
        const float x = s[r];
        float t;
        if constexpr (LOOK && POS == kPosTable)
          t = __builtin_fmaf(x, sc, nl4[e]) + tb[31 - qr];
        else if constexpr (LOOK && POS == kPosAlibi)
          t = __builtin_fmaf(-sl, __builtin_fabsf(dj - float(qr)),
                             __builtin_fmaf(x, sc, nl4[e]));
        else if constexpr (POS == kPosTable)
          t = __builtin_fmaf(x, sc, nl4[e]) + c;
        else
          t = __builtin_fmaf(x, sc, nl4[e]);
        if constexpr (MASK) t = uint32_t(qr - lo) <= span ? t : -kInf;
        const float p = __builtin_amdgcn_exp2f(t);
        float d = dp[r];
        if constexpr (DROP) {
          const uint32_t other =
              __builtin_amdgcn_update_dpp(0u, hb[r & 7], 0xb1, 0xf, 0xf, false);  // lane ^ 1
          const uint32_t bits = (lane & 1) == (q >> 1) ? hb[r & 7] : other;
          const float mult = (bits << low) >= thr ? up : 0.0f;
          pd[e] = p * mult;
          d = __builtin_fmaf(d, mult, dl4[e]);
        } else {
          pd[e] = p;
        }
        ds[e] = p * d;
      }
      pkp[2 * q] = pack_bf16x2(pd[0], pd[1]);
      pkp[2 * q + 1] = pack_bf16x2(pd[2], pd[3]);
      pkd[2 * q] = pack_bf16x2(ds[0], ds[1]);
      pkd[2 * q + 1] = pack_bf16x2(ds[2], ds[3]);
    }
  };

  if (work) {
#pragma unroll
    for (int st = 0; st < S::kStages; ++st) issue(uint32_t(st) * kStageKV);
  }
  if constexpr (POS != kPosAlibi) kr.take(kf, own, 0u);
  vr.take(vf, own, 0u);
  uint32_t boff = 0;
  if (work) {
    gemm::wait_vmcnt<(S::kStages - 1) * 5 * KS>();
    __syncthreads();
  }
  for (int h = h_a; work && h <= h_b; ++h) {
    if constexpr (POS == kPosTable) {
      __syncthreads();  // the previous head's table is read no more
      stage_bias(a, h, tab);
      __syncthreads();
      far_l = tab[0];
      far_r = tab[bias_entries(a.far) - 1];
    }
    if constexpr (POS == kPosAlibi) {
      sl = a.slopes[h] * kLog2e;
      bc.init(sl, sc, lane);
    }
    const int n_last = h == h_b ? n_b : t_hi;
    for (int first = h == h_a ? n_a : t_lo; first <= n_last; first += KS) {
      const int n = first + tg;
      const int i0 = n * kRows, i1 = i0 + kRows - 1;
      const bool some =
          n <= n_last && wk < L && ((i0 <= wk_hi + wl && i1 >= wk - wr) || wk < ns);
      if (some) {
        const f32x16 zero16 = {};
        const uint32_t pair = boff + tg * kPairKV;
        const char* const Q = ring + pair;
        const char* const D = Q + kTileBytes;
        const bool all = i1 < L && ((i1 <= wk + wl && i0 >= wk_hi - wr) || wk_hi < ns);
        using T_ = std::true_type;
        using F_ = std::false_type;
        float c = 0.0f;
        bool look = false, before = false;
        if constexpr (POS == kPosTable) {
          const bool left = wk + kCols - 1 - i0 <= -a.far, right = wk - i1 >= a.far;
          look = !left && !right;
          c = left ? far_l : far_r;
        }
        if constexpr (POS == kPosAlibi) {
          before = i1 <= wk;
          look = !(bc.ok && (before || i0 >= wk + kCols - 1));
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          f32x16 s, dp = zero16;
          if constexpr (!DROP) {  // dP from -delta, as in dq_kernel
            const float* nd = reinterpret_cast<const float*>(ring + pair + 2 * kTileBytes) + 64 +
                              32 * b + 4 * half;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 x = *reinterpret_cast<const f32x4*>(nd + 8 * q);
#pragma unroll
              for (int e = 0; e < 4; ++e) dp[4 * q + e] = x[e];
            }
          }
#pragma unroll
          for (int kc = 0; kc < 4; ++kc)
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.row(Q, b, kc), kf[kc],
                                                        kc == 0 ? zero16 : s, 0, 0, 0);
#pragma unroll
          for (int kc = 0; kc < 4; ++kc)
            dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.row(D, b, kc), vf[kc], dp, 0, 0, 0);
          uint32_t pkp[8], pkd[8];
          if constexpr (POS == kPosAlibi)
            if (!look) s = bc.add_half(s, b, float(jk - i0), before);
          if (POS != kPosNone && look) {
            if (all)
              grad(F_{}, T_{}, n, b, s, dp, 0.0f, pair, pkp, pkd);
            else
              grad(T_{}, T_{}, n, b, s, dp, 0.0f, pair, pkp, pkd);
          } else {
            if (all)
              grad(F_{}, F_{}, n, b, s, dp, c, pair, pkp, pkd);
            else
              grad(T_{}, F_{}, n, b, s, dp, c, pair, pkp, pkd);
          }
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const bf16x8 pf = chunk(pkp, cc), df = chunk(pkd, cc);
#pragma unroll
            for (int mb = 0; mb < 2; ++mb) {
              dv[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.trans(D, 2 * b + cc, mb), pf,
                                                               dv[mb], 0, 0, 0);
              dk[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fr.trans(Q, 2 * b + cc, mb), df,
                                                               dk[mb], 0, 0, 0);
            }
          }
        }
      }
      // the next stage landed, and every wave has read all of this one
      gemm::wait_vmcnt<(S::kStages - 2) * 5 * KS>();
      __syncthreads();
      issue(boff);
      boff = boff + kStageKV == S::kStages * kStageKV ? 0 : boff + kStageKV;
    }
  }
  // refills past the last tile may still be landing in this workgroup's LDS
  gemm::wait_vmcnt<0>();

  if constexpr (KS == 2) {
    float v[64];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        v[32 * i + r] = dk[i][r];
        v[32 * i + 16 + r] = dv[i][r];
      }
    if (!join_waves(v, ring, wave, lane)) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dk[i][r] = v[32 * i + r];
        dv[i][r] = v[32 * i + 16 + r];
      }
  }
  if (!own) return;
  if (splits > 1) {
    const int64_t row =
        sink_block ? ((int64_t(z) * a.sink_splits + split) * (a.n_heads / a.group) + hk) *
                             (a.sink_blocks * S::kOwn) + jk
                   : (int64_t(split) * (a.n_heads / a.group) + hk) * a.total + s0 + jk;
    float* p = (sink_block ? a.sink_part : a.kv_part) + row * (2 * kHeadDim) + 4 * half;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        *reinterpret_cast<f32x4*>(p + 32 * mb + 8 * q) =
            f32x4{dk[mb][4 * q], dk[mb][4 * q + 1], dk[mb][4 * q + 2], dk[mb][4 * q + 3]};
        *reinterpret_cast<f32x4*>(p + kHeadDim + 32 * mb + 8 * q) =
            f32x4{dv[mb][4 * q], dv[mb][4 * q + 1], dv[mb][4 * q + 2], dv[mb][4 * q + 3]};
      }
    return;
  }
  const int64_t t = s0 + jk;
  uint16_t* kp = a.dk + t * a.dk_tok + hk * a.dk_head + 4 * half;
  uint16_t* vp = a.dv + t * a.dv_tok + hk * a.dv_head + 4 * half;
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint2 w;
      w.x = pack_bf16x2(dk[mb][4 * q] * a.scale, dk[mb][4 * q + 1] * a.scale);
      w.y = pack_bf16x2(dk[mb][4 * q + 2] * a.scale, dk[mb][4 * q + 3] * a.scale);
      *reinterpret_cast<uint2*>(kp + 32 * mb + 8 * q) = w;
      w.x = pack_bf16x2(dv[mb][4 * q], dv[mb][4 * q + 1]);
      w.y = pack_bf16x2(dv[mb][4 * q + 2], dv[mb][4 * q + 3]);
      *reinterpret_cast<uint2*>(vp + 32 * mb + 8 * q) = w;
    }
}

// The splits' sums of a key row added up in order, 32 rows per workgroup, a thread 8 dims of dK
// and dV: first the rows of the sinks' blocks, where those are split, then the others.
__host__ __device__ __forceinline__ int join_sinks(const LocalArgs& a) {
  return a.sink_splits > 1 ? (a.n_seqs * a.sink_blocks << a.kb.shift) / 32 : 0;
}
__global__ __launch_bounds__(256) void kv_join_kernel(LocalArgs a, Blocks rows) {
  const int hk = blockIdx.y;
  const int hkv = a.n_heads / a.group;
  const int sink_rows = a.sink_blocks << a.kb.shift;
  const int n_sink = join_sinks(a);
  const int d = 8 * (threadIdx.x & 7);
  int z, s0, L, r, splits;
  const float* p;
  int64_t step;
  if (int(blockIdx.x) < n_sink) {
    z = int(blockIdx.x) / (sink_rows / 32);
    sequence(a, z, s0, L);
    r = int(blockIdx.x) % (sink_rows / 32) * 32 + (threadIdx.x >> 3);
    if (r >= L) return;
    splits = a.sink_splits;
    step = int64_t(hkv) * sink_rows;
    p = a.sink_part + (int64_t(z) * splits * step + int64_t(hk) * sink_rows + r) * (2 * kHeadDim);
  } else {
    if (!find_block(a, rows, int(blockIdx.x) - n_sink, z, s0, L, r)) return;
    r += threadIdx.x >> 3;
    if (r >= L || r < sink_rows) return;
    splits = a.splits;
    step = int64_t(hkv) * a.total;
    p = a.kv_part + (int64_t(hk) * a.total + s0 + r) * (2 * kHeadDim);
  }
  float k[8] = {}, v[8] = {};
  for (int i = 0; i < splits; ++i, p += step * (2 * kHeadDim)) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + d + e);
      const f32x4 y = *reinterpret_cast<const f32x4*>(p + kHeadDim + d + e);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        k[e + u] += x[u];
        v[e + u] += y[u];
      }
    }
  }
  const int64_t t = s0 + r;
  u32x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(k[2 * e] * a.scale, k[2 * e + 1] * a.scale);
  *reinterpret_cast<u32x4*>(a.dk + t * a.dk_tok + hk * a.dk_head + d) = w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
  *reinterpret_cast<u32x4*>(a.dv + t * a.dv_tok + hk * a.dv_head + d) = w;
}

}  // namespace

// How the backward's work is split: enough workgroups for 256 CUs to hold two each and some to
// spare, none of less than six steps; the sinks' key blocks into pieces of the others' length.
BwdPlan bwd_plan(int max_len, int n_seqs, int n_heads, int n_kv_heads, int64_t total, int wl,
                 int wr, int ns, int far) {
  BwdPlan p;
  Blocks whole;
  whole.init(total, n_seqs, max_len, 7);
  const int64_t full = whole.count;  // blocks of 128 rows of one head, about
  // (with a table's sums in LDS beside two KS = 2 stages a CU would hold one workgroup)
  p.ks = far > 0 ? 1 : pick_ks(full * n_heads);
  p.qb.init(total, n_seqs, max_len, p.ks == 2 ? 6 : 7);
  const int group = n_heads / n_kv_heads;
  p.kv_ks = pick_ks(full * n_kv_heads);
  const int kv_rows = 128 / p.kv_ks;
  p.kb.init(total, n_seqs, max_len, p.kv_ks == 2 ? 6 : 7);
  // A key block's query tiles are split where its workgroups would not fill the GPU's 512
  // places, into at least 6 steps each (split against whole, 12 heads on fewer key heads:
  // 1 x 2,048 on 4 heads 39.4 + 4.5 for the join, 84 us; 1 x 4,550 on 2 172 + 4.7, 346;
  // 1 x 777 on 1 19.3 + 6.2, 134).  Steps: 64 queries, KS of them at a time.
  const int64_t all = int64_t((max_len + kRows - 1) / kRows) * group / p.kv_ks + 1;
  const int64_t window =
      std::min<int64_t>(all, ((int64_t(wl) + wr + kv_rows) / kRows + 1) * group / p.kv_ks + 1);
  p.splits = int(std::max<int64_t>(1, std::min<int64_t>(512 / (full * n_kv_heads * p.kv_ks),
                                                        window / 6)));
  p.sink_blocks =
      window < all ? (std::min(ns, max_len) + kv_rows - 1) / kv_rows : 0;
  // (numbered for every sequence: where most are far shorter than their sinks, and beyond what a
  // launch holds, the sinks' blocks stay whole among the others)
  const int64_t sinks = int64_t(n_seqs) * p.sink_blocks;
  if (sinks > 4 * int64_t(p.kb.count) || sinks * n_kv_heads > (int64_t(1) << 22))
    p.sink_blocks = 0;
  const int64_t piece = std::max<int64_t>(6, window / p.splits);
  // (many sequences fill the GPU by themselves, and need no more than 256 MB of sums)
  const int64_t most = std::max<int64_t>(
      1, 4096 / (int64_t(n_seqs) * n_kv_heads * std::max(1, p.sink_blocks)));
  p.sink_splits = p.sink_blocks > 0
                      ? int(std::min({int64_t(64), most, (all + piece - 1) / piece}))
                      : 1;
  const int64_t row = 2 * kHeadDim;
  p.kv_part = p.splits > 1 ? int64_t(p.splits) * n_kv_heads * total * row : 0;
  p.sink_part = p.sink_splits > 1 ? int64_t(n_seqs) * p.sink_splits * n_kv_heads *
                                        p.sink_blocks * kv_rows * row
                                  : 0;
  p.bias_part = far > 0 ? int64_t(p.qb.count) * n_heads * (2 * far + 1) : 0;
  p.norms = 2 * int64_t(p.qb.count) * n_heads;
  return p;
}

hipError_t launch_local_bwd(const LocalArgs& a, bool wide, bool norms, hipStream_t st) {
  const bool table = a.bias != nullptr, grad = a.dbias != nullptr;
  const size_t tab = table ? size_t(bias_entries(a.far)) * 4 : 0;
  const size_t extra_q =
      tab * (grad ? 1 + kGradTables : 1) + (grad ? size_t(4) * kDiagFloats * 4 + 8 : 0);
  const int hkv = a.n_heads / a.group;
  if (norms) {
    const hipError_t e = launch_key_norm_max(a.k, a.k_tok, a.k_head, a.total, hkv,
                                             const_cast<float*>(a.kmax), st);
    if (e != hipSuccess) return e;
  }
  auto launch = [&](auto kernel, int64_t blocks, size_t lds) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(256), lds, st, a);
    return hipGetLastError();
  };
  auto launch_q = [&](auto kernel, int ks) {
    return launch(kernel, grid_blocks(a.qb.count, a.n_heads),
                  size_t(ks == 2 ? 4 : 3) * kPairQ + extra_q);
  };
  auto launch_kv = [&](auto kernel, int ks) {
    return launch(kernel, grid_blocks(kv_units(a), hkv) + (grad ? a.n_heads : 0),
                  size_t(ks == 2 ? 4 : 3) * kPairKV + tab);
  };
  auto run = [&](auto pos, auto drop) {
    constexpr int P = decltype(pos)::value;
    constexpr bool D = decltype(drop)::value;
    constexpr bool G = P == kPosTable;  // (a bias gradient only where there is a table)
    auto at = [&](auto w) {
      constexpr bool W = decltype(w)::value;
      hipError_t e;
      if (a.ks == 2)
        e = launch_q(dq_kernel<P, D, false, W, 2>, 2);
      else
        e = grad ? launch_q(dq_kernel<P, D, G, W, 1>, 1)
                 : launch_q(dq_kernel<P, D, false, W, 1>, 1);
      if (e != hipSuccess) return e;
      return a.kv_ks == 2 ? launch_kv(dkv_kernel<P, D, W, 2>, 2)
                          : launch_kv(dkv_kernel<P, D, W, 1>, 1);
    };
    return wide ? at(std::true_type{}) : at(std::false_type{});
  };
  auto pick = [&](auto pos) {
    return a.drop.on ? run(pos, std::true_type{}) : run(pos, std::false_type{});
  };
  hipError_t e = table ? pick(std::integral_constant<int, kPosTable>{})
                 : a.slopes != nullptr ? pick(std::integral_constant<int, kPosAlibi>{})
                                       : pick(std::integral_constant<int, kPosNone>{});
  if (e != hipSuccess) return e;
  if (a.splits > 1 || (a.sink_blocks > 0 && a.sink_splits > 1)) {
    Blocks rows;
    rows.init(a.total, a.n_seqs, a.max_len, 5);
    const int blocks = join_sinks(a) + (a.splits > 1 ? rows.count : 0);
    hipLaunchKernelGGL(kv_join_kernel, dim3(unsigned(blocks), unsigned(hkv)), dim3(256), 0, st, a,
                       rows);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace attn
}  // namespace g5moe
