// Attention with a sliding window, sink tokens, a bucketed relative position bias (or
// ALiBi) and dropout on the probabilities: the forward pass.
//
// For query i of a sequence of length L (positions inside the sequence)
//   visible keys  V(i) = { j < L : i - wl <= j <= i + wr  or  j < ns }
//   t_ij = scale q_i . k_j + bias_ij,  P = softmax of t over V(i)
//   O_i  = sum_j m_ij P_ij v_j,        lse_i = log sum_j exp t_ij
// with m_ij the dropout multiplier (1 without dropout), so the softmax is normalised by
// the undropped sum.  A row whose every visible term is -inf (a bias of -inf) gives O = 0
// and lse = -inf.
//
// Work split: one workgroup of four waves per (128 queries, head, sequence), a wave holding
// 32 queries; the 64-key tiles that any of the 128 queries sees (the sinks' tiles, then the
// window's) stream through a ring of three in LDS, filled by LDS DMA.  One pass over the
// keys with the running maximum and sum of the softmax, scores transposed (S^T = K Q^T) so
// that a query's statistics live in two lanes and the probabilities are the B operand of
// O^T += V^T P^T as they stand (attn_tile.h).  Per wave a tile is skipped (nothing of it is
// visible to the wave's queries), plain (all of it visible, the bias constant or linear), or
// takes the per-element path (MASK: an edge of the window, the sinks or the sequence; LOOK:
// the bias from the table, or ALiBi across the diagonal).
//
// What bounds it: the instructions of the softmax beside the products.  Counters, all SIMDs:
// 8 x 4,550 tokens, 12 heads, ALiBi: matrix units busy 32 % of the time, vector instructions
// issued 60 %, LDS reads 15 % without a bank conflict, 175 MB read from memory, 1.8 of 2 waves
// per SIMD.  A third wave per SIMD fits without the reads ahead (2 x 4,550, buckets: 199 us
// with two waves, 208 with three).
// Measured (12 heads; the formula's rate): ALiBi in a window of 512 + 512 with 16 sinks, 8 x
// 4,550 tokens, 190 us; buckets 2 x 4,550 203 us (625 TFLOP/s), 16 x 512 38 us, 777 tokens 15
// us; window of 1,024 + 1,024 over 1 x 9,000 111 us (517 TFLOP/s); ALiBi 8 x 4,550 304 us (most
// tiles are out of reach: all would take 600); a window over 77 tokens 6 us.
#include <algorithm>
#include <type_traits>

#include "attn_tile.h"

namespace g5moe {
namespace attn {
namespace {

constexpr int kPairBytes = 2 * kTileBytes;  // a K tile, then its V tile

template <int POS, bool DROP, bool WIDE, int KS>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2, 2)))
void local_fwd_kernel(LocalArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  using S = Split<KS>;
  constexpr int kStageBytes = KS * kPairBytes;
  char* const ring = smem;
  float* const tab = reinterpret_cast<float*>(smem + S::kStages * kStageBytes);

  int slot, hq;
  if (!block_of(blockIdx.x, a.qb.count, a.n_heads, slot, hq)) return;
  if (POS == kPosAlibi && a.kmax != nullptr && a.n_heads <= 64)
    hq = by_slope(a.slopes, a.n_heads, hq);
  zero_tail(a, a.o, a.o_tok, hq * a.o_head, slot, a.qb.count);
  int z, s0, L, q0;
  if (!find_block(a, a.qb, slot, z, s0, L, q0)) return;
  const int hk = hq / a.group;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int tg = S::tile(wave);
  const int wq = q0 + S::own(wave) * kCols;       // the wave's queries: wq .. wq_hi
  const int wq_hi = min(wq + kCols, L) - 1;
  const int iq = wq + col;
  const int wl = min(a.wl, L), wr = min(a.wr, L), ns = min(a.ns, L);
  // a negative scale is taken as its magnitude on negated queries (the same products)
  const float sc = __builtin_fabsf(a.sc);
  const float sl = POS == kPosAlibi ? a.slopes[hq] * kLog2e : 0.0f;

  bf16x8 qf[4];
  OwnRows qr;
  qr.request(a.q + int64_t(s0 + min(iq, L - 1)) * a.q_tok + hq * a.q_head, half);

  KeyTiles kt;
  TilePair<WIDE> tiles;
  tiles.init(ring, wave, lane, L, a.k_tok * 2, a.v_tok * 2);
  FragReader fr;
  fr.init(lane);
  const char* const kbase =
      reinterpret_cast<const char*>(a.k + int64_t(s0) * a.k_tok + hk * a.k_head);
  const char* const vbase =
      reinterpret_cast<const char*>(a.v + int64_t(s0) * a.v_tok + hk * a.v_head);
  // The next tile to load; past the last one it goes out again, into a buffer that no later
  // tile reads, so that every step issues the same number of loads.
  int n_is = 0;
  auto issue = [&](uint32_t boff) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < KS; ++g) {
      tiles.issue(kbase, vbase, __builtin_amdgcn_readfirstlane(n_is), boff + g * kPairBytes);
      n_is = n_is < kt.w_hi ? kt.next(n_is) : n_is;
    }
  };
  auto begin = [&](int reach) __attribute__((always_inline)) {
    kt.init(q0, min(q0 + S::kOwn, L) - 1, L, min(wl, reach), min(wr, reach),
            q0 - (ns - 1) > reach ? 0 : ns);
    n_is = kt.first();
#pragma unroll
    for (int st = 0; st < S::kStages; ++st) issue(uint32_t(st) * kStageBytes);
  };
  if constexpr (POS != kPosAlibi) begin(L);
  qr.take(qf, iq < L, a.sc < 0.0f ? 0x80008000u : 0u);
  if constexpr (POS == kPosAlibi) {
    // With the key norms, keys farther than `reach` from every query of the workgroup are left
    // out: their terms are below 2^-40 of the query's own key's, which it sees.
    int reach = L;
    if (a.kmax != nullptr) {
      OwnRows kr;
      kr.request(a.k + int64_t(s0 + min(iq, L - 1)) * a.k_tok + hk * a.k_head, half);
      bf16x8 kf[4];
      kr.take(kf, iq < L, 0u);
      float dot = 0.0f;
#pragma unroll
      for (int kc = 0; kc < 4; ++kc)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          dot = __builtin_fmaf(float(qf[kc][e]), float(kf[kc][e]), dot);
      dot += __shfl_xor(dot, 32, 64);
      __shared__ float red[2][4];
      float v[2] = {norm_max(qf), iq < L ? -sc * dot : -kInf};
      block_max(v, red, wave, lane);
      const float bound = sc * v[0] * key_norm(a, hk, s0, L, red, wave, lane);
      reach = alibi_reach(bound + v[1], sl, L);
    }
    begin(reach);
  }
  if constexpr (POS == kPosTable) {
    stage_bias(a, hq, tab);
    __syncthreads();
  }
  const float far_l = POS == kPosTable ? tab[0] : 0.0f;
  const float far_r = POS == kPosTable ? tab[bias_entries(a.far) - 1] : 0.0f;
  BiasChunk bc;
  if constexpr (POS == kPosAlibi) bc.init(sl, sc, lane);

  uint32_t rkey = 0, thr = 0;
  if constexpr (DROP) {
    rkey = dropout_row_key(uint32_t(s0 + iq) * uint32_t(a.n_heads) + uint32_t(hq),
                           a.drop.seed_lo, a.drop.seed_hi);
    thr = min(a.drop.thr, 65535u) << 16;  // p = 1: the scale is 0
  }

  f32x16 o[2] = {f32x16{}, f32x16{}};
  // what the exponents subtract, ms: the running maximum m (0 while every term was -inf).  A
  // bound of the row's terms in its place saves 3 % under ALiBi, but the probability of a row's
  // first key is exactly 1 only against the maximum itself; else its rounding to bf16 is the
  // larger part of a steep head's error (out 2.1e-3 against 2.3e-3, dq 2.4e-3 and 2.6e-3).
  float m = -kInf, ms = 0.0f, psum = 0.0f;
  f32x16 s[2];

  auto advance = [&](float mx) __attribute__((always_inline)) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx),
                                                     false, false);
    mx = __builtin_fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
    const float m_new = __builtin_fmaxf(m, mx);
    if (__ballot(m_new != m) != 0) {
      ms = m_new == -kInf ? 0.0f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m - ms);
      m = m_new;
      psum *= alpha;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[mb][r] *= alpha;
    }
  };
  // The softmax step: probabilities of the scores in s (PLAIN: scores to be scaled, the tile's
  // constant bias c to be added; else terms).
  uint32_t pk[2][8];
  auto softmax = [&](auto plain_c, int n, float c) __attribute__((always_inline)) {
    constexpr bool PLAIN = decltype(plain_c)::value;
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        mx = __builtin_fmaxf(__builtin_fmaxf(mx, s[b][r]), s[b][r + 1]);
    if constexpr (PLAIN)
      advance(POS == kPosTable ? __builtin_fmaf(mx, sc, c) : mx * sc);
    else
      advance(mx);
    const float sub = POS == kPosTable && PLAIN ? c - ms : -ms;
    const uint32_t jp = uint32_t(n * kRows + 4 * half) >> 1;
    float sum = 0.0f;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        float p[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float t = PLAIN ? __builtin_fmaf(s[b][r + e], sc, sub) : s[b][r + e] + sub;
          p[e] = __builtin_amdgcn_exp2f(t);
          sum += p[e];
        }
        if constexpr (DROP) {
          const uint32_t bits =
              dropout_pair_bits(rkey, jp + uint32_t(32 * b + 8 * (r >> 2) + (r & 3)) / 2);
          p[0] = uint16_t(bits) >= uint16_t(thr >> 16) ? p[0] : 0.0f;
          p[1] = bits >= thr ? p[1] : 0.0f;
        }
        pk[b][r >> 1] = pack_bf16x2(p[0], p[1]);
      }
    psum += sum;
  };
  // Per-element terms in place of the scores.
  auto terms = [&](auto mask_c, auto look_c, int n, float c) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_c)::value, LOOK = decltype(look_c)::value;
    const int j0 = n * kRows + 4 * half;   // the lane's first key
    const int lo = iq - wl - j0;           // window: tile offsets lo .. lo + span
    const uint32_t span = uint32_t(min(iq + wr, L - 1) - (iq - wl));
    const int sink = ns - j0;
    const float di = float(iq - j0);
    const float* tb = tab + (j0 - iq + a.far + kBiasPad);
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kr = 32 * b + 8 * (r >> 2) + (r & 3);
        float t;
        if constexpr (LOOK && POS == kPosTable)
          t = __builtin_fmaf(s[b][r], sc, tb[kr]);
        else if constexpr (LOOK && POS == kPosAlibi)
          t = __builtin_fmaf(-sl, __builtin_fabsf(di - float(kr)), s[b][r] * sc);
        else
          t = __builtin_fmaf(s[b][r], sc, c);
        if constexpr (MASK) t = (uint32_t(kr - lo) <= span || kr < sink) ? t : -kInf;
        s[b][r] = t;
      }
  };

  // Operands are read ahead: a tile's K fragments behind the previous tile's output product,
  // its V fragments before the softmax.
  uint32_t boff = 0;
  bf16x8 kf[2][4], vf[4][2];
  auto load_kf = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int kc = 0; kc < 4; ++kc)
#pragma unroll
      for (int b = 0; b < 2; ++b) kf[b][kc] = fr.row(ring + boff + tg * kPairBytes, b, kc);
  };
  // (behind the softmax where dropout and ALiBi take their registers)
  constexpr bool kLateV = DROP && POS == kPosAlibi;
  auto load_vf = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
        vf[c][mb] = fr.trans(ring + boff + tg * kPairBytes + kTileBytes, c, mb);
  };
  auto scores = [&]() __attribute__((always_inline)) {
    const f32x16 zero16 = {};
#pragma unroll
    for (int kc = 0; kc < 4; ++kc)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[b][kc], qf[kc],
                                                       kc == 0 ? zero16 : s[b], 0, 0, 0);
    if constexpr (!kLateV) load_vf();
  };
  auto turn = [&]() __attribute__((always_inline)) {
    if constexpr (kLateV) load_vf();
    // the next stage landed, and every wave has read all of this one
    gemm::wait_vmcnt<(S::kStages - 2) * 4 * KS>();
    __syncthreads();
    issue(boff);
    boff = boff + kStageBytes == S::kStages * kStageBytes ? 0 : boff + kStageBytes;
    load_kf();
  };
  auto output = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const bf16x8 pf = chunk(pk[c >> 1], c & 1);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
        o[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[c][mb], pf, o[mb], 0, 0, 0);
    }
  };
  using T_ = std::true_type;
  using F_ = std::false_type;

  // The wave's plain tiles: [all_lo, all_hi] or up to sink_hi are wholly visible, and of those
  // the ones up to before_hi or from after_lo have a bias of one kind.
  const bool any = wq < L;
  const int all_lo = any ? (max(wq_hi - wl, 0) + kRows - 1) / kRows : kNever;
  const int all_hi = (min(wq + wr, L - 1) + 1) / kRows - 1;
  const int sink_hi = any ? ns / kRows - 1 : -1;
  int before_hi = -1, after_lo = 0;
  if constexpr (POS == kPosTable) {
    before_hi = ((wq - a.far + 1) >> 6) - 1;
    after_lo = (wq_hi + a.far + kRows - 1) / kRows;
  }
  if constexpr (POS == kPosAlibi) {
    before_hi = bc.ok ? (wq + 1) / kRows - 1 : -1;
    after_lo = bc.ok ? (wq_hi + kRows - 1) / kRows : kNever;
  }

  int n = kt.first();
  if (tg == 1) n = kt.next(n);
  gemm::wait_vmcnt<(S::kStages - 1) * 4 * KS>();
  __syncthreads();
  load_kf();
  for (int left = kt.count(); left > 0;) {
    // a run of plain tiles of one kind, without branches
    const bool before = POS != kPosNone && n <= before_hi;
    int hi = n >= all_lo && n <= all_hi ? all_hi : n <= sink_hi ? sink_hi : -1;
    if (POS != kPosNone) hi = before ? min(hi, before_hi) : n >= after_lo ? hi : -1;
    if (n < kt.s_end) hi = min(hi, kt.s_end - 1);
    const int run = min(hi >= n ? (hi - n) / KS + 1 : 0, (left - tg + KS - 1) / KS);
    if (run > 0) {
      const float c = before ? far_l : far_r;
      float d = float(iq - n * kRows);
      for (int i = 0; i < run; ++i) {
        scores();
        if constexpr (POS == kPosAlibi) {
          bc.add(s, d, before);
          d -= float(KS * kRows);
        }
        softmax(T_{}, n + i * KS, c);
        turn();
        output();
      }
      left -= run * KS;
      n += (run - 1) * KS;
    } else {
      const int j0 = n * kRows, j1 = j0 + kRows - 1;
      // what the wave's queries see of the tile
      const bool some =
          left > tg && any && ((j0 <= wq_hi + wr && j1 >= wq - wl) || j0 < ns);
      if (some) {
        scores();
        const bool all = (n >= all_lo && n <= all_hi) || n <= sink_hi;
        const bool look = POS != kPosNone && !before && !(n >= after_lo);
        const float c = before ? far_l : far_r;
        if constexpr (POS == kPosAlibi)
          if (!look) bc.add(s, float(iq - j0), before);
        if (!look)
          terms(T_{}, F_{}, n, c);
        else if (all)
          terms(F_{}, T_{}, n, c);
        else
          terms(T_{}, T_{}, n, c);
        softmax(F_{}, n, c);
      }
      turn();
      if (some) output();
      left -= KS;
    }
#pragma unroll
    for (int g = 0; g < KS; ++g) n = kt.next(n);
  }
  // refills past the last tile may still be landing in this workgroup's LDS
  gemm::wait_vmcnt<0>();

  float l = psum + __shfl_xor(psum, 32, 64);
  if constexpr (KS == 2) {
    // both waves' sums at the larger of their maxima
    float* const other = reinterpret_cast<float*>(ring);
    __syncthreads();
    other[wave * 64 + lane] = m;
    __syncthreads();
    const float top = __builtin_fmaxf(m, other[(wave ^ 2) * 64 + lane]);
    const float f = m == -kInf ? 0.0f : __builtin_amdgcn_exp2f(m - top);
    m = top;
    float v[33];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      v[r] = o[0][r] * f;
      v[16 + r] = o[1][r] * f;
    }
    v[32] = l * f;
    if (!join_waves(v, ring + 1024, wave, lane)) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      o[0][r] = v[r];
      o[1][r] = v[16 + r];
    }
    l = v[32];
  }
  if (iq < L) {
    const float inv = l == 0.0f ? 0.0f : (DROP ? a.drop.scale : 1.0f) / l;
    uint16_t* op = a.o + int64_t(s0 + iq) * a.o_tok + hq * a.o_head + 4 * half;
    uint16_t* low = a.o_low + (int64_t(s0 + iq) * a.n_heads + hq) * kHeadDim + 4 * half;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float x0 = o[mb][4 * q] * inv, x1 = o[mb][4 * q + 1] * inv;
        const float x2 = o[mb][4 * q + 2] * inv, x3 = o[mb][4 * q + 3] * inv;
        uint2 w;
        w.x = pack_bf16x2(x0, x1);
        w.y = pack_bf16x2(x2, x3);
        *reinterpret_cast<uint2*>(op + 32 * mb + 8 * q) = w;
        if (a.o_low != nullptr) {
          const uint2 rest = {pack_rest_bf16x2(x0, x1, w.x), pack_rest_bf16x2(x2, x3, w.y)};
          *reinterpret_cast<uint2*>(low + 32 * mb + 8 * q) = rest;
        }
      }
    if (a.lse != nullptr && half == 0)
      a.lse[int64_t(hq) * a.total + s0 + iq] = l == 0.0f ? -kInf : (m + __builtin_log2f(l)) * kLn2;
  }
}

__global__ __launch_bounds__(256) void zero_behind_kernel(LocalArgs a) {
  zero_tail(a, a.o, a.o_tok, int64_t(blockIdx.y) * a.o_head, int(blockIdx.x), int(gridDim.x));
}

}  // namespace

// Of 128-row blocks; a CU holds two workgroups.  Two waves to 32 rows are worth their loads only
// where the GPU is not filled (12 heads, one wave against two): forward 1 x 777 13.2, 9.9 us;
// dq_kernel 1 x 2,048 46, 39; but 4 x 1,100 44, 49; 8 x 4,550 825, 926.
int pick_ks(int64_t blocks128) { return blocks128 < 256 ? 2 : 1; }

hipError_t launch_zero_behind(const LocalArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(zero_behind_kernel, dim3(16, unsigned(a.n_heads)), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_local_fwd(const LocalArgs& a, bool wide, hipStream_t st) {
  const dim3 grid(unsigned(grid_blocks(a.qb.count, a.n_heads)));
  if (a.kmax != nullptr) {
    const hipError_t e = launch_key_norm_max(a.k, a.k_tok, a.k_head, a.total,
                                             a.n_heads / a.group, const_cast<float*>(a.kmax), st);
    if (e != hipSuccess) return e;
  }
  auto launch = [&](auto kernel, int stages, int ks) {
    const size_t lds = size_t(stages * ks) * kPairBytes +
                       (a.bias != nullptr ? bias_entries(a.far) * 4 : 0);
    hipLaunchKernelGGL(kernel, grid, dim3(256), lds, st, a);
    return hipGetLastError();
  };
  auto pick = [&](auto pos, auto drop) {
    constexpr int P = decltype(pos)::value;
    constexpr bool D = decltype(drop)::value;
    if (wide)
      return a.ks == 2 ? launch(local_fwd_kernel<P, D, true, 2>, 2, 2)
                       : launch(local_fwd_kernel<P, D, true, 1>, 3, 1);
    return a.ks == 2 ? launch(local_fwd_kernel<P, D, false, 2>, 2, 2)
                     : launch(local_fwd_kernel<P, D, false, 1>, 3, 1);
  };
  auto with_drop = [&](auto pos) {
    return a.drop.on ? pick(pos, std::true_type{}) : pick(pos, std::false_type{});
  };
  if (a.bias != nullptr) return with_drop(std::integral_constant<int, kPosTable>{});
  if (a.slopes != nullptr) return with_drop(std::integral_constant<int, kPosAlibi>{});
  return with_drop(std::integral_constant<int, kPosNone>{});
}

}  // namespace attn
}  // namespace g5moe
