// Building blocks of the attention kernels with options (attention_local.hip,
// attention_bwd.hip): 64-row tiles of two bf16 matrices streamed through a ring in LDS,
// the fragment reads of such a tile, the set of keys that a query sees, the relative
// position bias and the dropout bits.  Device code for gfx950 only.
//
// MFMA layout (v_mfma_f32_32x32x16_bf16).  The streamed tile gives the 64 rows of the
// product (two halves of 32), the wave's own 32 rows its columns: lane l holds column
// l % 32 and, in element 4q + u of half b, row 32b + 8q + 4(l / 32) + u.  A following
// product over the tile's rows takes these elements as its B operand without moving
// them: elements 8(c % 2) .. + 8 of half c / 2 are the k-chunk of rows 16c .. + 16, with
// row 4(l / 32) + (e & 3) + 8(e >> 2) in place e; its A operand, the tile transposed, is
// read in the same order.
//
// LDS layout.  A row is 128 bytes, 8 chunks of 16.  Chunk c of row r is stored at
// c ^ swz(r), swz(r) = 4 (bit 1 of r) + (bits 2, 3 of r).  A row read (16 lanes at 16
// consecutive rows, one chunk) then falls on all 64 banks: swz takes its eight values once
// over the eight rows of each parity.  A transposing read (four rows r, 4 chunks each) does
// too: rows of one parity differ in bit 1, so in the half of the row they use.
#pragma once

#include "gemm_common.h"

namespace g5moe {
namespace attn {

using gemm::bf16x8;
using gemm::f32x16;
using gemm::i16x4;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kHeadDim = 64;
constexpr int kCols = 32;                        // the wave's own rows
constexpr int kRows = 64;                        // rows of a streamed tile
constexpr int kRowBytes = kHeadDim * 2;
constexpr int kTileBytes = kRows * kRowBytes;    // 8 KB
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_inff();
constexpr int kNever = 0x7fffffff;
// Entries of the bias table in LDS beyond the largest distance on either side: a tile that
// reaches within that distance of the wave's rows holds distances up to 95 past it.
constexpr int kBiasPad = 96;

enum Pos { kPosNone = 0, kPosAlibi = 1, kPosTable = 2 };

__device__ __forceinline__ uint32_t swz(int r) {
  return uint32_t(((r >> 1) & 1) * 4 + ((r >> 2) & 3));
}

typedef __attribute__((address_space(3))) i16x4* lds_i16x4_p;
// ds_read_b64_tr_b16: within each 16-lane group the lanes' 64-bit chunks form a 16 x 4
// matrix (lane k's chunk is row k), and lane i receives element i % 4 of rows i / 4,
// 4 + i / 4, 8 + i / 4 and 12 + i / 4.
__device__ __forceinline__ i16x4 read_tr(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4_p>(
      uintptr_t((__attribute__((address_space(3))) const char*)p)));
}

// LDS DMA of 64 x 16 bytes: with a base in scalar registers and a 32-bit offset per lane
// (all five wait states between a VALU write of the base and its use are waited here, four
// instructions per tile), and with a 64-bit address per lane.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_dma16_u(const char* base, uint32_t voff, uint32_t lds) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  const uint64_t u = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(p)))) |
                     uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(uint32_t(p >> 32)))) << 32;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(voff), "s"(u), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory", "m0");
}
__device__ __forceinline__ void lds_dma16_v(const char* addr, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :: "v"(addr), "s"(__builtin_amdgcn_readfirstlane(lds))
               : "memory", "m0");
}
#pragma clang diagnostic pop

// How the four waves of a workgroup share its work: KS = 1: each has 32 own rows, all of them
// every tile; KS = 2: two waves share 32 own rows and take every second tile each, and their
// sums are joined at the end.  The second needs twice the loads per product, and halves the
// smallest unit of work: for launches of few workgroups.
template <int KS>
struct Split {
  static constexpr int kOwn = 4 / KS * kCols;             // own rows per workgroup
  static constexpr int kStages = KS == 1 ? 3 : 2;         // of KS tile pairs each
  static __device__ __forceinline__ int own(int wave) { return KS == 1 ? wave : wave & 1; }
  static __device__ __forceinline__ int tile(int wave) { return KS == 1 ? 0 : wave >> 1; }
};

// The DMA of one 64-row tile of each of two matrices by four waves (tile a, then tile b
// 8 KB behind): instruction i of a wave fills rows 8 (4i + wave) .. + 8, so four instructions
// per wave and call.  Rows past `rows` in the sequence's last tile repeat its last row.
// WIDE: a row stride too large for 32-bit offsets inside a tile.
template <bool WIDE>
struct TilePair {
  int64_t sa, sb;        // bytes between rows
  uint32_t lds;          // ring + wave * 1024
  int last;              // number of the sequence's last tile
  int lastrow;           // its last row
  int row[2];
  uint32_t ch;           // the lane's byte inside a row
  uint32_t oa[2][2], ob[2][2];  // [last tile][instruction]

  __device__ __forceinline__ void init(const char* ring, int wave, int lane, int len, int64_t sa_,
                                       int64_t sb_) {
    sa = sa_;
    sb = sb_;
    lds = gemm::lds_addr(ring) + uint32_t(wave) * 1024;
    last = (len - 1) / kRows;
    lastrow = (len - 1) % kRows;
    const int lr = lane >> 3;
    ch = (uint32_t(lane & 7) ^ swz(8 * (wave & 1) + lr)) * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      row[i] = (4 * i + wave) * 8 + lr;
      const int rl = min(row[i], lastrow);
      oa[0][i] = uint32_t(row[i]) * uint32_t(sa) + ch;
      ob[0][i] = uint32_t(row[i]) * uint32_t(sb) + ch;
      oa[1][i] = uint32_t(rl) * uint32_t(sa) + ch;
      ob[1][i] = uint32_t(rl) * uint32_t(sb) + ch;
    }
  }
  // Tile n of the matrices at a and b (their row 0) into the ring at byte boff.
  __device__ __forceinline__ void issue(const char* a, const char* b, int n, uint32_t boff) const {
    const char* ta = a + int64_t(n) * kRows * sa;
    const char* tb = b + int64_t(n) * kRows * sb;
    const bool is_last = n == last;
    const uint32_t dst = lds + boff;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (WIDE) {
        const int r = is_last ? min(row[i], lastrow) : row[i];
        lds_dma16_v(ta + r * sa + ch, dst + i * 4096);
        lds_dma16_v(tb + r * sb + ch, dst + kTileBytes + i * 4096);
      } else {
        lds_dma16_u(ta, is_last ? oa[1][i] : oa[0][i], dst + i * 4096);
        lds_dma16_u(tb, is_last ? ob[1][i] : ob[0][i], dst + kTileBytes + i * 4096);
      }
    }
  }
};

// Fragment addresses of a tile, per lane.
struct FragReader {
  int rowoff;      // the lane's row read: row col, chunk kc at ((2 kc + half) ^ rsw) * 16
  uint32_t rsw;
  int half;
  int tr[2][2];    // [dim half mb][hi]: transposing read of rows 8 hi + 4 half + (0..3)

  __device__ __forceinline__ void init(int lane) {
    const int col = lane & 31;
    half = lane >> 5;
    rowoff = col * kRowBytes;
    rsw = swz(col);
    const int vk = (lane & 15) >> 2;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi) {
        const int r = 8 * hi + 4 * half + vk;
        const uint32_t c = uint32_t(4 * mb + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1));
        tr[mb][hi] = r * kRowBytes + int((c ^ swz(r)) * 16) + 8 * (lane & 1);
      }
  }
  // A operand: rows 32 b + col, head dims 16 kc + 8 half .. + 8
  __device__ __forceinline__ bf16x8 row(const char* tile, int b, int kc) const {
    return *reinterpret_cast<const bf16x8*>(tile + rowoff + 32 * b * kRowBytes +
                                            ((uint32_t(2 * kc + half)) ^ rsw) * 16);
  }
  // A operand, transposed: head dims 32 mb + col over the rows of chunk c in the order of
  // the accumulator elements
  __device__ __forceinline__ bf16x8 trans(const char* tile, int c, int mb) const {
    const char* p = tile + 16 * c * kRowBytes;
    const i16x4 vv[2] = {read_tr(p + tr[mb][0]), read_tr(p + tr[mb][1])};
    return __builtin_bit_cast(bf16x8, vv);
  }
};

// The wave's own rows as a B operand (head dims 16 kc + 8 half .. + 8): requested, so that
// other loads go out behind them, and taken later, when they have landed, so that no wait for
// them falls into the tile loop.  Zeros where !ok (the request still has to be in bounds).
struct OwnRows {
  u32x4 w[4];
  __device__ __forceinline__ void request(const uint16_t* p, int half) {
#pragma unroll
    for (int kc = 0; kc < 4; ++kc)
      w[kc] = *reinterpret_cast<const u32x4*>(p + 16 * kc + 8 * half);
  }
  __device__ __forceinline__ void take(bf16x8 (&f)[4], bool ok, uint32_t flip) {
#pragma unroll
    for (int kc = 0; kc < 4; ++kc) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[kc][e] = ok ? w[kc][e] ^ flip : 0u;
      asm volatile("" : "+v"(w[kc]));
      f[kc] = __builtin_bit_cast(bf16x8, w[kc]);
    }
  }
};

// A 32-row block's accumulator elements packed to bf16: rows 16c .. + 16 as a B operand.
__device__ __forceinline__ bf16x8 chunk(const uint32_t (&pk)[8], int c) {
  const u32x4 raw = {pk[4 * c + 0], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]};
  return __builtin_bit_cast(bf16x8, raw);
}

// The ALiBi bias of a tile wholly on one side of the wave's rows as one more 16-deep chunk
// of the score product, in units of raw scores: tile rows [r, r, r, 1, 1, 1, 0, 0] (r the
// row's offset in the tile, exact in bf16) against columns [+-u1, +-u2, +-u3, c1, c2, c3,
// 0, 0], where u1 + u2 + u3 = slope / scale and c1 + c2 + c3 = the column's constant are
// bf16 splits, exact to fp32 precision.  Usable for finite ratios of slope to scale.
struct BiasChunk {
  bool ok;
  float u;
  u32x4 kx[2];
  uint32_t qu[3];
  static __device__ __forceinline__ float bf16r(float x) { return float(__bf16(x)); }
  // sl: slope, sc: scale, both times log2(e)
  __device__ __forceinline__ void init(float sl, float sc, int lane) {
    const int half = lane >> 5, col = lane & 31;
    ok = __builtin_amdgcn_readfirstlane(
             int(sc != 0.0f && __builtin_fabsf(sl) < __builtin_fabsf(sc) * 0x1p60f)) != 0;
    u = ok ? sl / sc : 0.0f;
    const uint32_t half0 = half == 0 ? 0xffffffffu : 0u;
    const float u1 = bf16r(u), u2 = bf16r(u - u1), u3 = bf16r(u - u1 - u2);
    qu[0] = pack_bf16x2(u1, u2) & half0;
    qu[1] = pack_bf16x2(u3, 0.0f) & half0;
    qu[2] = 0x80008000u & half0;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float r = float(32 * b + col);
      kx[b] = u32x4{pack_bf16x2(r, r) & half0, pack_bf16x2(r, 1.0f) & half0,
                    pack_bf16x2(1.0f, 1.0f) & half0, 0u};
    }
  }
  // The scores s of half b of the tile with -u |own - row| added: d = own - (the tile's
  // first row), the tile before the wave's rows (own >= row everywhere) or after them.
  __device__ __forceinline__ f32x16 add_half(const f32x16& s, int b, float d, bool before) const {
    const float c = before ? -u * d : u * d;
    const uint32_t sign = before ? 0u : qu[2];
    const float c1 = bf16r(c), c2 = bf16r(c - c1), c3 = bf16r(c - c1 - c2);
    const u32x4 q = {qu[0] ^ sign,
                     (qu[1] ^ (sign & 0xffffu)) | (__float_as_uint(c1) & 0xffff0000u),
                     pack_bf16x2(c2, c3), 0u};
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kx[b]),
                                                   __builtin_bit_cast(bf16x8, q), s, 0, 0, 0);
  }
  __device__ __forceinline__ void add(f32x16* s, float d, bool before) const {
#pragma unroll
    for (int b = 0; b < 2; ++b) s[b] = add_half(s[b], b, d, before);
  }
};

// How blocks of 2^shift rows of the packed sequences are numbered: per > 0: that many for every
// sequence (those past its end unused), sequence z's from z per; per = 0: sequence z's from
// cu[z] / 2^shift + z, which leaves room for every block of the ones before, whatever their
// lengths, and at most one number of each sequence unused.  The host, which does not know the
// lengths, takes the one of fewer numbers: the first for sequences of about max_len.
struct Blocks {
  int shift, per, count;
  __host__ __device__ void init(int64_t total, int n_seqs, int max_len, int shift_) {
    shift = shift_;
    per = (max_len - 1) / (1 << shift) + 1;
    const int64_t packed = (total >> shift) + n_seqs;
    if (int64_t(per) * n_seqs > packed) per = 0;
    count = per > 0 ? per * n_seqs : int(packed);
  }
  __device__ __forceinline__ int first(int z, int s0) const {
    return per > 0 ? z * per : (s0 >> shift) + z;
  }
};
// Kernel arguments of the attention with options, forward and backward.
struct LocalArgs {
  const uint16_t *q, *k, *v, *dout;
  uint16_t* o;                      // forward: written; backward: read
  uint16_t* o_low;                  // what o's rounding left over, [total, n_heads, 64], or nullptr
  uint16_t *dq, *dk, *dv;
  const int32_t* cu;                // [n_seqs + 1]
  int64_t q_tok, k_tok, v_tok, o_tok, do_tok, dq_tok, dk_tok, dv_tok;  // element strides
  int64_t q_head, k_head, v_head, o_head, do_head, dq_head, dk_head, dv_head;
  int n_seqs, n_heads, group;
  float sc;                         // softmax_scale * log2(e)
  float scale;                      // softmax_scale
  const float* slopes;              // [n_heads] or nullptr
  const void* bias;                 // [n_buckets, n_heads], bf16 or fp32, or nullptr
  const int32_t* bucket_of;         // [2 far + 1]: bucket of key minus query position + far
  int bias_bf16, n_buckets, far;
  float* lse;                       // [n_heads, total]; natural log
  float* nl;                        // backward: -lse * log2(e), [n_heads, total]
  float* delta;                     // backward: -dout . o, [n_heads, total]
  uint32_t* rowkey;                 // backward with dropout: the rows' keys, [n_heads, total]
  float* part;                      // backward: bias sums per workgroup of dq_kernel
  void* dbias;                      // backward: [n_buckets, n_heads] or nullptr
  int wl, wr, ns;                   // window (large = unlimited), first tokens always visible
  // with ALiBi, for leaving out tiles whose probabilities vanish, or nullptr: the largest key
  // norm of each 64-token block [n_kv_heads, ceil(total / 64)], and (backward) the largest
  // query norm and the largest -lse log2(e) of each block of queries [n_heads, qb.count]
  const float* kmax;
  float2* qmax;
  Blocks qb;                        // of dq_kernel and the forward
  int ks, kv_ks;                    // Split of the kernels over queries and over keys
  // backward: the splits of a key block's query tiles (of the sinks' blocks) and their sums
  Blocks kb;
  int splits, sink_blocks, sink_splits;
  float *kv_part, *sink_part;
  int64_t total;
  int max_len;                      // sequences are not computed past it
  DropoutParams drop;
};

// The workgroup's (x, head) of nx x heads, from a one-dimensional grid of grid_blocks()
// workgroups, id the number of this one: consecutive workgroups go to the eight XCDs in turn,
// so runs of kRun blocks x of one head are given to one XCD, whose L2 then serves their common
// tiles (runs of 1, 8 and 32: 8 x 4,550 tokens dq 817, 809, 818 us, dkv 1,048, 1,041, 1,052;
// windows in ragged batches, whose work is less even, dq 118, 118, 131).  False: nothing to do.
constexpr int kXcds = 8;
constexpr int kRun = 8;
__device__ __forceinline__ bool block_of(uint32_t id, int nx, int heads, int& x, int& h) {
  const uint32_t j = id / kXcds;
  const uint32_t item = ((j / kRun) * kXcds + id % kXcds) * kRun + j % kRun;
  x = int(item % uint32_t(nx));
  h = int(item / uint32_t(nx));
  return h < heads;
}
inline int64_t grid_blocks(int64_t nx, int64_t heads) {
  constexpr int64_t unit = kXcds * kRun;
  return (nx * heads + unit - 1) / unit * unit;
}
// Head number r by rising ALiBi slope, so by falling work (the reach falls with the slope), so
// that the launch does not end on its longest workgroups.  Up to 64 heads.
__device__ __forceinline__ int by_slope(const float* slopes, int heads, int r) {
  const int lane = threadIdx.x & 63;
  const float own = lane < heads ? slopes[lane] : kInf;
  const float key = own > 0.0f ? own : 0.0f;  // no reach
  int rank = 0;
  for (int j = 0; j < heads; ++j) {
    const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(key), j));
    rank += other < key || (other == key && j < lane) ? 1 : 0;
  }
  return __builtin_ctzll(__ballot(lane < heads && rank == r));
}

// Sequence z's first token and length, clamped to [0, total] and max_len: a malformed
// cu_seqlens cannot move an access outside the buffers.
__device__ __forceinline__ void sequence(const LocalArgs& a, int z, int& s0, int& L) {
  const int total = int(a.total);
  s0 = __builtin_amdgcn_readfirstlane(min(max(a.cu[z], 0), total));
  L = __builtin_amdgcn_readfirstlane(min(min(max(a.cu[z + 1], s0), total) - s0, a.max_len));
}

// Number `slot`'s sequence z, its first token s0 and length L, and the block's first row in
// it; false where the number is unused.  Packed numbering: one load of cu_seqlens per 63
// sequences, lane i holds sequence base + i, whose starts rise with i.  Positions clamped as by
// sequence().
__device__ __forceinline__ bool find_block(const LocalArgs& a, const Blocks& nb, int slot, int& z,
                                           int& s0, int& L, int& row) {
  const int shift = nb.shift;
  if (nb.per > 0) {
    z = slot / nb.per;
    sequence(a, z, s0, L);
    row = (slot % nb.per) << shift;
    return row < L;
  }
  const int lane = threadIdx.x & 63;
  const int total = int(a.total);
  int base = 0;
  for (;;) {
    const int i = base + lane;
    const int c = min(max(a.cu[min(i, a.n_seqs)], 0), total);
    const bool starts = i < a.n_seqs && (c >> shift) + i <= slot;
    const uint64_t m = __ballot(starts);
    if ((m >> 63) != 0) {  // lane 63 is the next round's first
      base += 63;
      continue;
    }
    const int n = __builtin_popcountll(m);
    if (n == 0) return false;  // (only a cu_seqlens that does not begin at 0)
    z = base + n - 1;
    s0 = __builtin_amdgcn_readlane(c, n - 1);
    L = min(max(__builtin_amdgcn_readlane(c, n), s0) - s0, a.max_len);
    row = (slot - (s0 >> shift) - z) << shift;
    return row >= 0 && row < L;
  }
}

// KS = 2: the accumulators of waves 2 and 3 added to those of waves 0 and 1, by way of LDS
// (N x 256 bytes per wave pair at buf).  Every wave calls it; true for those that hold the sum.
template <int N>
__device__ __forceinline__ bool join_waves(float (&v)[N], char* buf, int wave, int lane) {
  float* const p = reinterpret_cast<float*>(buf) + (wave & 1) * N * 64 + lane;
  __syncthreads();
  if (wave >= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i * 64] = v[i];
  }
  __syncthreads();
  if (wave >= 2) return false;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += p[i * 64];
  return true;
}

// Largest norm of the wave's own 32 rows (every lane).
__device__ __forceinline__ float norm_max(const bf16x8 (&f)[4]) {
  float ss = 0.0f;
#pragma unroll
  for (int kc = 0; kc < 4; ++kc)
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(float(f[kc][e]), float(f[kc][e]), ss);
  ss += __shfl_xor(ss, 32, 64);
  return __builtin_sqrtf(ss);
}

// v[i] maximised over the workgroup's 256 lanes.
template <int N>
__device__ __forceinline__ void block_max(float (&v)[N], float (*red)[4], int wave, int lane) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int bit = 32; bit >= 1; bit >>= 1) v[i] = __builtin_fmaxf(v[i], __shfl_xor(v[i], bit, 64));
  __syncthreads();  // red is read no more
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) red[i][wave] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] = __builtin_fmaxf(__builtin_fmaxf(red[i][0], red[i][1]),
                           __builtin_fmaxf(red[i][2], red[i][3]));
}

// Largest key norm over the 64-token blocks that cover a sequence.
__device__ __forceinline__ float key_norm(const LocalArgs& a, int hk, int s0, int L,
                                          float (*red)[4], int wave, int lane) {
  const float* p = a.kmax + int64_t(hk) * ((a.total + 63) / 64);
  float km[1] = {0.0f};
  for (int i = (s0 >> 6) + int(threadIdx.x); i <= ((s0 + L - 1) >> 6); i += 256)
    km[0] = __builtin_fmaxf(km[0], p[i]);
  block_max(km, red, wave, lane);
  return km[0];
}

// The distance from which ALiBi's slope sl (times log2(e)) puts 2^(top - sl distance) below
// 2^-40; L where there is none (also for an infinite or NaN top).  The terms left out fall
// geometrically from there: together they are below 2^-39 / (1 - 2^-sl), and a reach within a
// sequence of length L means sl > 40 / L, so below L 2^-43: 2^-24, the rounding of one fp32
// term, for a million tokens.
__device__ __forceinline__ int alibi_reach(float top, float sl, int L) {
  const float w = (top + 40.0f) / sl;
  return __builtin_amdgcn_readfirstlane(sl > 0.0f && w < float(L) ? max(int(w) + 1, 0) : L);
}

// Rows behind the last sequence, [cu[n_seqs], total), of one head of a bf16 tensor: zeros, the
// work of 256-thread workgroups x = 0 .. nx - 1.
__device__ __forceinline__ void zero_tail(const LocalArgs& a, uint16_t* p, int64_t tok,
                                          int64_t head_off, int x, int nx) {
  const int end = max(a.cu[a.n_seqs], 0);
  for (int64_t r = int64_t(end) + int64_t(x) * 32 + (threadIdx.x >> 3); r < a.total;
       r += int64_t(nx) * 32)
    *reinterpret_cast<u32x4*>(p + r * tok + head_off + 8 * (threadIdx.x & 7)) = u32x4{0, 0, 0, 0};
}

// The head's bias table in LDS, times log2(e): entry x holds the bias at distance
// x - kBiasPad - far (key minus query position), clamped to +-far.
__device__ __forceinline__ void stage_bias(const LocalArgs& a, int h, float* tab) {
  const int n = 2 * a.far + 1;
  for (int x = threadIdx.x; x < n + 2 * kBiasPad; x += 256) {
    const int b = min(max(a.bucket_of[min(max(x - kBiasPad, 0), n - 1)], 0), a.n_buckets - 1);
    const int64_t at = int64_t(b) * a.n_heads + h;
    const float v = a.bias_bf16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(a.bias)[at])
                                : static_cast<const float*>(a.bias)[at];
    tab[x] = v * kLog2e;
  }
}

// LDS floats of the bias table.
__host__ __device__ constexpr int bias_entries(int far) { return 2 * far + 1 + 2 * kBiasPad; }

// The tiles that hold a key visible to queries [q_lo, q_hi] of a sequence of length L, in
// order: the sinks' [0, s_end), then [w_lo, w_hi].
struct KeyTiles {
  int s_end, w_lo, w_hi;
  __device__ __forceinline__ void init(int q_lo, int q_hi, int L, int wl, int wr, int ns) {
    const int sink_tiles = (min(ns, L) + kRows - 1) / kRows;
    w_lo = max(q_lo - wl, 0) / kRows;
    w_hi = max(min(q_hi + wr, L - 1) / kRows, sink_tiles - 1);
    s_end = min(sink_tiles, w_lo);
  }
  __device__ __forceinline__ int first() const { return s_end > 0 ? 0 : w_lo; }
  __device__ __forceinline__ int next(int n) const { return n + 1 == s_end ? w_lo : n + 1; }
  __device__ __forceinline__ int count() const { return s_end + w_hi - w_lo + 1; }
};

// The largest norm of each 64-token block of each head of k (attention.hip).
}  // namespace attn
hipError_t launch_key_norm_max(const uint16_t* k, int64_t tok, int64_t head, int64_t total,
                               int n_heads, float* out, hipStream_t st);
namespace attn {

// Zeros in the rows of out behind the last sequence.
hipError_t launch_zero_behind(const LocalArgs& a, hipStream_t st);
// Split of a launch over blocks of 128 own rows.
int pick_ks(int64_t blocks128);
// wide: a token stride of a streamed matrix of 2^24 elements or more.
hipError_t launch_local_fwd(const LocalArgs& a, bool wide, hipStream_t st);
// norms: a.kmax is to be written first.
hipError_t launch_local_bwd(const LocalArgs& a, bool wide, bool norms, hipStream_t st);
// The splits of the key/value gradients and the floats of the backward's buffers (far: the bias
// table's largest distance, 0 without a table).
struct BwdPlan {
  int ks, kv_ks;
  Blocks qb, kb;
  int splits, sink_blocks, sink_splits;
  int64_t kv_part, sink_part, bias_part, norms;
};
BwdPlan bwd_plan(int max_len, int n_seqs, int n_heads, int n_kv_heads, int64_t total, int wl,
                 int wr, int ns, int far);

}  // namespace attn
}  // namespace g5moe
