// Paged attention over the KV cache in 4 bits (format: mx4.h): prefill and
// decode, the formula, chunk statistics and bits of attn_impl.h's kernels over
// a cache of the values the codes stand for. Instantiated per activation type
// in attn_mx4_{bf16,f16}.hip.
//
// Every code becomes an exact 16-bit float (one conversion per two elements,
// the block's scale included) in the lane that feeds it to a matrix
// instruction or writes it to LDS, so scores and weighted V are the 16-bit
// MFMA chains of attn_impl.h in the same order. Scores are computed transposed
// (keys as the MFMA's rows, query rows as its columns): lane (kg, row i =
// lane % 16) gets keys 8 kg .. 8 kg + 7 of each 32-key step from two MFMAs
// whose key rows are pi(i) = 8 (i / 4) + 4 h + i % 4, h = 0, 1, which is its
// operand of the weighted-V MFMA: the weights never leave its registers.
//
// Two kernels:
//   attn_mx4_rows16_kernel  16 query rows a workgroup (decode, short prompts).
//     Bound by the cache's bytes, so its four waves take different key tiles of
//     a chunk and share nothing but the chunk's maxima and integer sums.
//   attn_mx4_prompt_kernel  128 query rows, or 64 (prompts). Bound by vector
//     arithmetic, so a key tile is unpacked once for the four waves.
#pragma once

#include "attn_impl.h"
#include "mx4.h"

namespace fxpr {
namespace attn {
namespace m4 {

using mx4::u32x2;

struct Mx4Args {
  AttnArgs a;  // (k, v and their strides unused)
  const uint8_t* kc;  // K codes, V codes, K scales, V scales
  const uint8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  uint32_t c_blk, c_slot, c_head, s_blk, s_slot, s_head;  // bytes
  float vlim;  // |x| below which the rounding constant quantises x (kRoundF)
  uint32_t by_group, by_heads, by_reqs;  // ceil(2^32 / x) of the group, kv heads and requests (see quotient)
};

// x / d with m = ceil(2^32 / d): exact while x d < 2^32 (the excess of m over
// 2^32 / d is below 1, so the product is off by less than x / 2^32, and x / d is
// at least 1 / d from the next integer). The host checks the ranges; d = 1 has
// m = 0. (An integer division by a variable is some 30 instructions, and a
// decode workgroup has only 8 key tiles to spread its start over.)
__host__ __device__ __forceinline__ uint32_t reciprocal(uint32_t d) {
  return d <= 1 ? 0u : uint32_t(((uint64_t(1) << 32) + d - 1) / d);
}
__device__ __forceinline__ uint32_t quotient(uint32_t x, uint32_t m) { return m == 0 ? x : __umulhi(x, m); }

// row_info (attn_impl.h) by quotient().
__device__ __forceinline__ RowInfo row_at(const Mx4Args& m, int g, int q_start, int q_len, int ctx, int seq_len, int row) {
  const AttnArgs& a = m.a;
  RowInfo ri;
  const int rows_total = q_len * a.group;
  const int rr = row < rows_total ? row : 0;
  const int i = int(quotient(uint32_t(rr), m.by_group));
  ri.token = q_start + i;
  ri.valid = row < rows_total && ri.token >= 0 && ri.token < a.num_tokens;
  if (!ri.valid) ri.token = 0;
  ri.head = g * a.group + (rr - i * a.group);
  ri.qpos = ctx + i;
  ri.kend = a.causal ? min(seq_len, ri.qpos + 1) : seq_len;
  ri.kstart = a.window > 0 ? max(0, ri.qpos - a.window + 1) : 0;
  return ri;
}

// The request of a workgroup whose place in the launch order is request slot x
// of a pass (a row tile, a key split) over the requests: slot x + pass, around.
// Workgroups go to the XCDs and to the shader engines of an XCD in turn,
// whatever those still hold, so in a grid of requests x passes one request's
// workgroups would all go to the same engines and the longest request's engines
// end last (prompts of 2048, 1547, 1083 and 1534 tokens, 8 kv heads: each
// request on one engine of every XCD). Every second pass: the passes of two
// requests then reach all four engines too.
__device__ __forceinline__ int turned(const Mx4Args& m, int x, int pass) {
  const uint32_t v = uint32_t(x + (pass >> 1));
  return int(v - quotient(v, m.by_reqs) * uint32_t(m.a.num_requests));
}

// quant() (fxp_device.h) with its saturating conversion in place. The compiler
// waits for an MFMA result before its own instructions name the result's
// registers, not before an asm statement does, and an element of a result that
// nothing reads (a workgroup of few rows) is a free register while the MFMA still
// writes it; here the register is one that the rounding has just written.
__device__ __forceinline__ int32_t cvt_sat(float integral) {
  asm("v_cvt_i32_f32 %0, %0" : "+v"(integral));
  return __builtin_bit_cast(int32_t, integral);
}
template <int BITS> __device__ __forceinline__ int64_t quant(float s) {
  const float r = __builtin_rintf(s);
  if constexpr (BITS == 64) {
    return __builtin_fabsf(r) < 2147483648.0f ? static_cast<int64_t>(cvt_sat(r)) : quant_i64(s);
  } else {
    const int32_t v = cvt_sat(r);
    return BITS == 16 ? (v < -32768 ? -32768 : (v > 32767 ? 32767 : v)) : v;
  }
}

// The rounding constant of the fast quantisation: for |x| 2^f < 2^22,
// fl(x 2^f + 1.5 2^23) (exact product, one rounding, spacing 1, an even
// constant) has the bits of RNE(x 2^f) + kRound.
constexpr float kRoundF = 12582912.0f;
constexpr uint32_t kRound = 0x4B400000u;

// Sets of 64 query rows of a prompt's workgroup (16 a wave): two where their
// sums fit a wave's registers (but for the folded ones, which a chunk's end
// alone needs and takes from scratch). Two sets take a key tile's unpacking, LDS
// reads and barrier once: four prompts of up to 2048 tokens 208 us, one set 253
// (235 with a third workgroup per CU); 8 x 512 new tokens over 16000 keys 2.26 ms
// against 2.70.
constexpr int row_sets(int bits, int head_dim) { return bits != 64 && head_dim <= 128 ? 2 : 1; }

// Host plan of a launch.
struct Mx4Plan {
  int splits = 1;            // key splits of the 16-row workgroups (every splits-th chunk)
  int pq_splits = 1;         // of the prompts' workgroups (chunks dealt evenly)
  bool prompt = false;       // requests of kPrefillRows rows or more in the prompts' workgroups
  int sets = 1;              // row sets of the prompts' workgroups (at most row_sets())
  int tok_cap = 0;           // AttnArgs::tok_cap
};

typedef const __attribute__((address_space(4))) int32_t* ConstI32;

// Scale words of a row: D / 32 bytes.
template <int D> struct Scales {
  static constexpr int N = (D / 32 + 3) / 4;
  uint32_t w[N];
};
template <int D> __device__ __forceinline__ Scales<D> load_scales(const uint8_t* p) {
  Scales<D> s;
  if constexpr (D == 64) {
    s.w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if constexpr (D == 128) {
    s.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    s.w[0] = v[0];
    s.w[1] = v[1];
  }
  return s;
}
// A lane group's units of a row: D / 8 bytes.
template <int D> struct Units {
  uint32_t w[D / 32];
};
template <int D> __device__ __forceinline__ Units<D> load_units(const uint8_t* p) {
  Units<D> u;
  if constexpr (D == 64) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    u.w[0] = v[0];
    u.w[1] = v[1];
  } else {
#pragma unroll
    for (int j = 0; j < D / 32; j += 4) {
      const u32x4 v = reinterpret_cast<const u32x4*>(p)[j / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u.w[j + i] = v[i];
    }
  }
  return u;
}

// LDS rows of 16-byte chunks, chunk c of row r at slot c ^ swz(r).
template <int D> struct Lds {
  static constexpr int ROWB = D * 2, TILEB = TILE * ROWB;
  static __device__ __forceinline__ int vswz(int r) { return DmaGeom<D>::swz(r); }
  static __device__ __forceinline__ int kswz(int r) { return PDmaGeom<D>::kswz(r); }
};

__device__ __forceinline__ u32x4 lds_load16(const unsigned char* p) { return *reinterpret_cast<const u32x4*>(p); }
__device__ __forceinline__ void lds_store16(unsigned char* p, u32x4 v) { *reinterpret_cast<u32x4*>(p) = v; }
__device__ __forceinline__ u32x2 lds_load_tr8(const unsigned char* p) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(p)));
}

// Over the 16 lanes of a row, all of them getting the result: rotations within
// the row as operands of the operation itself.
template <int N> __device__ __forceinline__ int row_ror(int x) {
  return __builtin_amdgcn_update_dpp(0, x, 0x120 + N, 0xf, 0xf, false);
}
__device__ __forceinline__ float row16_max(float x) {
  auto step = [](float v, int y) { return fmaxf(v, __uint_as_float(uint32_t(y))); };
  x = step(x, row_ror<8>(int(__float_as_uint(x))));
  x = step(x, row_ror<4>(int(__float_as_uint(x))));
  x = step(x, row_ror<2>(int(__float_as_uint(x))));
  return step(x, row_ror<1>(int(__float_as_uint(x))));
}
__device__ __forceinline__ uint32_t row16_sum(uint32_t x) {
  x += uint32_t(row_ror<8>(int(x)));
  x += uint32_t(row_ror<4>(int(x)));
  x += uint32_t(row_ror<2>(int(x)));
  return x + uint32_t(row_ror<1>(int(x)));
}
__device__ __forceinline__ uint64_t row16_sum(uint64_t x) {
  auto turn = [](uint64_t v, auto n) {
    constexpr int N = decltype(n)::value;
    return (uint64_t(uint32_t(row_ror<N>(int(uint32_t(v >> 32))))) << 32) | uint32_t(row_ror<N>(int(uint32_t(v))));
  };
  x += turn(x, std::integral_constant<int, 8>{});
  x += turn(x, std::integral_constant<int, 4>{});
  x += turn(x, std::integral_constant<int, 2>{});
  return x + turn(x, std::integral_constant<int, 1>{});
}

// A workgroup barrier that orders LDS but waits for no global load in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Orders a wave's LDS writes before its other lanes' reads (the LDS serves a
// wave's accesses in order).
__device__ __forceinline__ void lds_wave_order() {
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");
}

// The paged cache as the kernels address it: 16-key granules, each within one
// page (pages hold 16, 32, ... keys), their block-table entries by scalar
// loads. Keys past the sequence read its last one (their scores are masked),
// table and block indices are clamped into range, so inconsistent metadata
// cannot address outside the cache.
struct Pager {
  ConstI32 row;
  int last_key, last_block, max_blocks, ps_shift, page_mask;
  __device__ __forceinline__ int granule(int g) const { return min(g, last_key >> 4); }
  // the table entry of (clamped) granule g
  __device__ __forceinline__ int entry(int g) const {
    return row[min((16u * uint32_t(g)) >> ps_shift, uint32_t(max_blocks - 1))];
  }
  // the same per lane (a vector load), granules of a chunk: any beyond the
  // sequence too (a clamped entry of the table row, never used)
  __device__ __forceinline__ int entry_at(int g) const {
    return reinterpret_cast<const int32_t*>((uint64_t)row)[min((16u * uint32_t(g)) >> ps_shift, uint32_t(max_blocks - 1))];
  }
  __device__ __forceinline__ uint32_t block(int e) const { return uint32_t(e < 0 ? 0 : min(e, last_block)); }
  // byte offset of granule g's first row
  __device__ __forceinline__ uint64_t offset(int g, int e, uint32_t blk, uint32_t slot, uint32_t head_off) const {
    return uint64_t(block(e)) * blk + uint64_t(uint32_t((16 * g) & page_mask)) * slot + head_off;
  }
  // the largest row offset (row index times slot) within granule g that lies in
  // the sequence: a lane takes the smaller of its own and this, so rows past the
  // sequence read bytes of its last row (their keys are masked)
  __device__ __forceinline__ uint32_t limit(int g, uint32_t slot) const {
    return uint32_t(min(last_key - 16 * g, 15)) * slot;
  }
};

template <class A> __device__ __forceinline__ Pager make_pager(const A& a, int r, int seq_len) {
  Pager p;
  p.row = (ConstI32)(a.bt + int64_t(r) * a.sbt);
  p.last_key = max(seq_len, 1) - 1;
  p.last_block = int(a.num_blocks - 1 < 0x7fffffff ? a.num_blocks - 1 : 0x7fffffff);
  p.max_blocks = a.max_blocks;
  p.ps_shift = a.ps_shift;
  p.page_mask = a.page_size - 1;
  return p;
}

// ---------------------------------------------------------------------------
// 16 query rows. Wave w takes tiles w and w + 4 of a chunk: K fragments go
// from global memory straight into the score MFMAs, V rows through a 32-key
// LDS stage of the wave's own (unpacked, then read transposed). Per chunk two
// barriers: the row maxima, and the waves' integer partial sums, which are
// added in any order to the same bits (attn_impl.h's waves split them by d
// instead). Loads run a phase ahead: a chunk's V goes out before its scores,
// the next chunk's K before the weights (with up to 4 rows behind them, where
// the registers of a third workgroup per CU are worth more).
//
// NE: the workgroup has up to 4 NE rows (a decode step has as many as the GQA
// group, often 4). The products are in the plain layout (query rows as the
// MFMA's rows), row p as MFMA row 4 (p % 4) + p / 4: lane group kg then has rows
// kg, kg + 4, .. in its result registers e = 0, 1, .., and with 4 rows only
// e = 0 holds any. The softmax and the sums run over NE of the 4 registers (the
// transposed layout of the prompts' kernel has no register to leave out: 102 us
// for 64 requests up to 8192 keys, where the weights cross LDS here).
//
// FAST (the same bits): no softcap or ALiBi and a positive scale, so a score is
// fl(dot * scale) and the chunk maximum fl(max(dot) * scale); sums by the
// rounding constant (a weight is at most 1; a tile whose weighted V leaves the
// constant's range is added exactly).
template <int BITS, int D, int MAXE> struct Rows16Lds {
  using AccT = typename AccOf<BITS>::T;
  // A wave's V stage: key row r at r * PITCH + (r / 8) * 32 bytes. The padding
  // keeps the banks apart of the four rows (of 32 bytes each, two row groups of
  // 8) that half a wave's transposing read takes and of the rows that its
  // writes go to, and every d block and chunk is a constant away from one
  // address (an XOR swizzle takes a register for each).
  static constexpr int PITCH = Lds<D>::ROWB + 64;
  static constexpr int STAGEB = 32 * PITCH + 3 * 32;
  static constexpr int ROWS = 4 * MAXE;
  static constexpr int PARTB = ROWS * D * int(sizeof(AccT));        // its partial sums, in the stage's place
  static constexpr int WAVEB = STAGEB > PARTB ? STAGEB : PARTB;
  static constexpr int VP = TILE + 8;                               // pitch of a row of weights
  unsigned char stage[4][WAVEB];
  uint16_t p[4][ROWS * VP];
  float red_m[2][4][QROWS];  // (by the chunk's parity: no third barrier)
  AccT red_d[4][QROWS];
};

// A workgroup's request and rows.
struct Rows16 {
  int r, g, q_start, q_len, seq_len, ctx, row0;
};

template <int DT, int BITS, int D, bool SPLIT, bool FAST, int NE, int MAXE>
__device__ __forceinline__ void rows16_body(const Mx4Args& m, const Rows16& w, Rows16Lds<BITS, D, MAXE>& lds, int ent) {
  const AttnArgs& a = m.a;
  using TR = Traits<DT>;
  using T = typename TR::T;
  using AccT = typename AccOf<BITS>::T;
  using RL = Rows16Lds<BITS, D, MAXE>;
  constexpr int QS = D / 32, DBLK = D / 16, NT = CT / 4;
  constexpr int TPR = 64 / NE;       // threads per row in the sums over the waves
  constexpr int VPT = NE * D / 64;   // elements of the row per thread
  const int tid = threadIdx.x, lane = tid & 63, kg = lane >> 4, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  unsigned char* stage = lds.stage[wave];
  uint16_t* pw = lds.p[wave];
  auto ws_row = [&](int64_t token) { return a.tok_cap > 0 ? int64_t(w.r) * a.tok_cap + (token - w.q_start) : token; };
  const int rows_total = w.q_len * a.group;
  const int i_min = int(quotient(uint32_t(w.row0), m.by_group));
  const int i_max = int(quotient(uint32_t(min(rows_total - 1, w.row0 + 4 * NE - 1)), m.by_group));
  const int hi = a.causal ? min(w.seq_len, w.ctx + i_max + 1) : w.seq_len;
  const int lo = a.window > 0 ? max(0, w.ctx + i_min - a.window + 1) : 0;
  const int t_lo = lo / TILE;
  const int t_hi = hi > lo ? (hi + TILE - 1) / TILE : t_lo;
  const int c_first = t_lo / CT;
  int c_end = t_hi > t_lo ? (t_hi + CT - 1) / CT : c_first;
  if constexpr (SPLIT) c_end = min(c_end, a.chunk_slots);
  // this workgroup's chunks: every stride-th
  const int stride = SPLIT ? a.num_splits : 1;
  const int c_lo = c_first + (SPLIT ? int(blockIdx.z) : 0);
  auto row_of = [&](int p) { return row_at(m, w.g, w.q_start, w.q_len, w.ctx, w.seq_len, w.row0 + p); };

  if (SPLIT && blockIdx.z == 0 && tid < 4 * NE) {
    const RowInfo ri = row_of(tid);
    if (ri.valid) {
      int* cr = a.crange + 2 * (ws_row(ri.token) * a.num_heads + ri.head);
      cr[0] = c_first;
      cr[1] = c_end;
    }
  }
  if (SPLIT && c_lo >= c_end) return;  // uniform

  const Pager pager = make_pager(a, w.r, w.seq_len);
  const uint32_t ch = uint32_t(w.g) * m.c_head, sh = uint32_t(w.g) * m.s_head;
  auto live_lo = [&](int c) { return max(c * CT, t_lo); };
  auto live_hi = [&](int c) { return min(c * CT + CT, t_hi); };
  // the wave's tile u (0, 1) of chunk c, moved onto a live one (whose loads are
  // in flight anyway) where it is none
  auto tile_of = [&](int c, int u) { return min(max(c * CT + wave + 4 * u, live_lo(c)), live_hi(c) - 1); };

  // The byte offsets of a chunk's 32 granules, a lane each, from their table
  // entries (loaded a chunk ahead; the first ones by the caller).
  uint32_t oc_lo, oc_hi, os_lo, os_hi;
  auto offsets = [&](int c) __attribute__((always_inline)) {
    const int gq = 32 * c + (lane & 31);
    const uint64_t oc = pager.offset(gq, ent, m.c_blk, m.c_slot, ch), os = pager.offset(gq, ent, m.s_blk, m.s_slot, sh);
    oc_lo = uint32_t(oc);
    oc_hi = uint32_t(oc >> 32);
    os_lo = uint32_t(os);
    os_hi = uint32_t(os >> 32);
  };
  auto at_lane = [](uint32_t x, int l) { return uint32_t(__builtin_amdgcn_readlane(int(x), l)); };
  // A granule of the wave's tile: uniform bases and limits (Pager) of its code
  // and scale rows.
  struct Granule {
    uint64_t c, s;
    uint32_t cl, sl;
  };
  constexpr uint32_t kLastUnit = 3 * (D / 8);
  auto granule = [&](int c, int t, int q) __attribute__((always_inline)) {
    const int gq = pager.granule(4 * t + q), l = gq - 32 * c;
    Granule x;
    x.c = (uint64_t(at_lane(oc_hi, l)) << 32) | at_lane(oc_lo, l);
    x.s = (uint64_t(at_lane(os_hi, l)) << 32) | at_lane(os_lo, l);
    x.cl = pager.limit(gq, m.c_slot) + kLastUnit;
    x.sl = pager.limit(gq, m.s_slot);
    return x;
  };
  // K: lane (kg, i16) has row i16 of the granule, units kg. V: lane l has row
  // l / 4, units l % 4.
  const uint32_t kc_off = i16 * m.c_slot + kg * (D / 8), ks_off = i16 * m.s_slot;
  const uint32_t vc_off = uint32_t(lane >> 2) * m.c_slot + (lane & 3) * (D / 8), vs_off = uint32_t(lane >> 2) * m.s_slot;
  Units<D> kb[NT][4], vb[NT][4];
  Scales<D> kbs[NT][4], vbs[NT][4];
  auto load_k = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const Granule x = granule(c, tile_of(c, u), q);
        kb[u][q] = load_units<D>(m.kc + x.c + min(kc_off, x.cl));
        kbs[u][q] = load_scales<D>(m.ks + x.s + min(ks_off, x.sl));
      }
  };
  auto load_v = [&](int c, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const Granule x = granule(c, tile_of(c, u), q);
      vb[u][q] = load_units<D>(m.vc + x.c + min(vc_off, x.cl));
      vbs[u][q] = load_scales<D>(m.vs + x.s + min(vs_off, x.sl));
    }
  };
  if (c_lo < c_end) {
    offsets(c_lo);
    load_k(c_lo);
  }

  // Q as the A operand: lane row i16 is row i16 / 4 + 4 (i16 % 4).
  u32x4 qf[QS];
  {
    const RowInfo ri = row_of((i16 >> 2) + 4 * (i16 & 3));
    const bool use = ri.valid && (i16 & 3) < NE;
    const T* qbase = static_cast<const T*>(a.q) + ri.token * a.sq_t + int64_t(ri.head) * a.sq_h;
#pragma unroll
    for (int j = 0; j < QS; ++j)
      qf[j] = use ? *reinterpret_cast<const u32x4*>(qbase + 32 * j + 8 * kg) : u32x4{0u, 0u, 0u, 0u};
  }
  // The lane's rows kg + 4 e of the results: visible keys (none outside the request).
  int ks[NE], ke[NE], qp[NE];
  float slope[NE];
  int all_lo = 0, all_hi = 0x7fffffff;  // keys that every row of the lane sees
#pragma unroll
  for (int e = 0; e < NE; ++e) {
    const RowInfo ri = row_of(kg + 4 * e);
    ks[e] = ri.valid ? ri.kstart : 0x7fffffff;
    ke[e] = ri.valid ? ri.kend : 0;
    qp[e] = ri.qpos;
    slope[e] = !FAST && a.alibi ? a.alibi[ri.head] : 0.0f;
    // (rows outside the request see no key and are never stored: they count as
    // seeing everything)
    all_lo = max(all_lo, ri.valid ? ri.kstart : 0);
    all_hi = min(all_hi, ri.valid ? ri.kend : 0x7fffffff);
  }
  auto tile_whole = [&](int t) -> bool {
    return __builtin_amdgcn_ballot_w64(!(all_lo <= t * TILE && t * TILE + TILE <= all_hi)) == 0;
  };

  // LDS addresses of the V stage: where the lane writes (row lane / 4, chunk
  // lane % 4; chunk 4 j + lane % 4 is 64 j on, the second granule 16 rows), and
  // its transposing reads (keys 8 kg + j / 4 + 4 h, columns 4 (j % 4) of d block
  // 0, j = lane % 16; d block b is 32 b on).
  unsigned char* vst = stage + (lane >> 2) * RL::PITCH + (lane >> 5) * 32 + (lane & 3) * 16;
  const unsigned char* vld = stage + (8 * kg + (i16 >> 2)) * RL::PITCH + kg * 32 + (i16 & 3) * 8;
  // the weights' rows: written by result rows, read as the A operand's
  uint16_t* pst = pw + kg * RL::VP + i16;
  const uint16_t* pld = pw + ((i16 >> 2) + 4 * ((i16 & 3) < NE ? (i16 & 3) : 0)) * RL::VP + 8 * kg;

  // the thread's part of the sums: row tid / TPR, elements my_d ..
  const int my_row = tid / TPR, my_d = VPT * (tid % TPR);
  float M = -__builtin_inff();
  AccT Dn = 0, W[VPT];
#pragma unroll
  for (int v = 0; v < VPT; ++v) W[v] = 0;

  if (c_lo < c_end) {
    for (int c = c_lo, par = 0;; c += stride, par ^= 1) {
      const int ta = live_lo(c), te = live_hi(c);
      const bool more = c + stride < c_end;  // uniform
      load_v(c, 0);
      if constexpr (MAXE > 1) load_v(c, 1);
      if (more) ent = pager.entry_at(32 * (c + stride) + (lane & 31));
      auto next_k = [&]() __attribute__((always_inline)) {
        if (more) {
          offsets(c + stride);
          load_k(c + stride);
        }
      };

      // the wave's tiles: dots (FAST) or scores, for the lane's rows and keys
      // 16 q + i16 of the tile, -inf where masked
      float sc[NT][4][NE], mx[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) mx[e] = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int t = c * CT + wave + 4 * u;
        const bool live = t >= ta && t < te;  // uniform
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < QS; ++j)
            acc = TR::mma(qf[j], mx4::unpack8<DT>(kb[u][q].w[j], mx4::scale_of<DT>(kbs[u][q].w[j / 4], j % 4)), acc);
#pragma unroll
          for (int e = 0; e < NE; ++e) {
            float x = acc[e];
            if constexpr (!FAST) {
              x = __fmul_rn(x, a.scale_log2);
              if (a.softcap_log2 > 0.0f) x = softcapped(x, a.softcap_log2);
              if (a.alibi) x = x + slope[e] * static_cast<float>(t * TILE + 16 * q + i16 - qp[e]);
            }
            sc[u][q][e] = x;
          }
        }
        if (!live || !tile_whole(t)) {  // uniform
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < NE; ++e) {
              const int key = t * TILE + 16 * q + i16;
              sc[u][q][e] = (live && key >= ks[e] && key < ke[e]) ? sc[u][q][e] : -__builtin_inff();
            }
        }
#pragma unroll
        for (int e = 0; e < NE; ++e)
          mx[e] = fmaxf(fmaxf(mx[e], fmaxf(sc[u][0][e], sc[u][1][e])), fmaxf(sc[u][2][e], sc[u][3][e]));
      }
      if constexpr (MAXE > 1) next_k();
      else load_v(c, 1);

      // the chunk's row maxima: the row's 16 lanes, then the waves
      float(&rm)[4][QROWS] = lds.red_m[par];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        mx[e] = row16_max(mx[e]);
        if constexpr (FAST) mx[e] = __fmul_rn(mx[e], a.scale_log2);
        if (i16 == 0) rm[wave][kg + 4 * e] = mx[e];
      }
      lds_barrier();
      float mrow[NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        const int p = kg + 4 * e;
        const float x = fmaxf(fmaxf(rm[0][p], rm[1][p]), fmaxf(rm[2][p], rm[3][p]));
        mrow[e] = x != -__builtin_inff() ? x : 0.0f;  // no key: pin to 0
      }

      // weights and weighted V of the wave's tiles. FAST: the sums carry
      // kRound per added term, taken out below.
      AccT den[NE], wv[DBLK][NE];
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        den[e] = 0;
#pragma unroll
        for (int b = 0; b < DBLK; ++b) wv[b][e] = 0;
      }
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const int t = c * CT + wave + 4 * u;
        if (t >= ta && t < te) {  // uniform
          lds_wave_order();
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < NE; ++e) {
              const float x = FAST ? __fmul_rn(sc[u][q][e], a.scale_log2) : sc[u][q][e];
              const float wt = __builtin_amdgcn_exp2f(x - mrow[e]);
              if constexpr (FAST)  // (the maximum: NaN counts as 0)
                den[e] = AccT(uint32_t(den[e]) + __float_as_uint(fmaxf(__builtin_fmaf(wt, a.fxp_scale, kRoundF), kRoundF)));
              else
                den[e] = wadd<BITS>(den[e], quant<BITS>(__fmul_rn(wt, a.fxp_scale)));
              pst[4 * e * RL::VP + 16 * q] = FAST ? uint16_t(p_pack2<DT>(wt, wt)) : Io<DT>::store(wt);
            }
          f32x4 acc[DBLK];
#pragma unroll
          for (int b = 0; b < DBLK; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int j = 0; j < QS; ++j)
                lds_store16(vst + (q * (16 * RL::PITCH + 64) + 64 * j),
                            mx4::unpack8<DT>(vb[u][2 * s + q].w[j],
                                             mx4::scale_of<DT>(vbs[u][2 * s + q].w[j / 4], j % 4)));
            lds_wave_order();
            const u32x4 pa = *reinterpret_cast<const u32x4*>(pld + 32 * s);
#pragma unroll
            for (int b = 0; b < DBLK; ++b) {
              const u32x2 lo2 = lds_load_tr8(vld + 32 * b);
              const u32x2 hi2 = lds_load_tr8(vld + (4 * RL::PITCH + 32 * b));
              acc[b] = TR::mma(pa, u32x4{lo2[0], lo2[1], hi2[0], hi2[1]}, acc[b]);
            }
            lds_wave_order();
          }
          if constexpr (FAST) {
            auto term = [&](float x) { return __float_as_uint(__builtin_fmaf(x, a.fxp_scale, kRoundF)); };
            float vmax = 0.0f;
#pragma unroll
            for (int e = 0; e < NE; ++e) {
              den[e] = AccT(uint32_t(den[e]) - 4u * kRound);
#pragma unroll
              for (int b = 0; b < DBLK; ++b) {
                vmax = __builtin_elementwise_maximum(vmax, __builtin_fabsf(acc[b][e]));
                wv[b][e] = AccT(uint32_t(wv[b][e]) + term(acc[b][e]));
              }
            }
            if (__builtin_amdgcn_ballot_w64(!(vmax < m.vlim)) != 0) {  // uniform: out of the constant's range
#pragma unroll
              for (int b = 0; b < DBLK; ++b)
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                  const AccT without = AccT(uint32_t(wv[b][e]) - term(acc[b][e]));
                  wv[b][e] = AccT(uint32_t(wadd<BITS>(without, quant<BITS>(__fmul_rn(acc[b][e], a.fxp_scale)))) + kRound);
                }
            }
          } else {
#pragma unroll
            for (int b = 0; b < DBLK; ++b)
#pragma unroll
              for (int e = 0; e < NE; ++e)
                wv[b][e] = wadd<BITS>(wv[b][e], quant<BITS>(__fmul_rn(acc[b][e], a.fxp_scale)));
          }
        }
      }

      // the waves' partial sums to LDS, rows of D, the 16-element group x of row p
      // at x ^ (p % 4): lane (kg, i16) holds elements 16 b + i16 of its rows
#pragma unroll
      for (int e = 0; e < NE; ++e) {
        den[e] = AccT(row16_sum(typename std::make_unsigned<AccT>::type(den[e])));
        if (i16 == 0) lds.red_d[wave][kg + 4 * e] = den[e];
        AccT* p = reinterpret_cast<AccT*>(stage) + (kg + 4 * e) * D + i16;
#pragma unroll
        for (int b = 0; b < DBLK; ++b) p[16 * (b ^ kg)] = wv[b][e];
      }
      lds_barrier();
      const RowInfo mine = row_of(my_row);
      if (mine.valid) {
        const AccT cd = wadd<BITS>(wadd<BITS>(lds.red_d[0][my_row], lds.red_d[1][my_row]),
                                   wadd<BITS>(lds.red_d[2][my_row], lds.red_d[3][my_row]));
        const float cm = fmaxf(fmaxf(rm[0][my_row], rm[1][my_row]), fmaxf(rm[2][my_row], rm[3][my_row]));
        const int at = my_row * D + (my_d ^ ((my_row & 3) << 4));
        AccT cw[VPT];
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
          cw[v] = 0;
#pragma unroll
          for (int x = 0; x < 4; ++x) cw[v] = wadd<BITS>(cw[v], reinterpret_cast<const AccT*>(lds.stage[x])[at + v]);
          if constexpr (FAST) cw[v] = AccT(uint32_t(cw[v]) - uint32_t(te - ta) * kRound);
        }
        if constexpr (SPLIT) {
          const int64_t slot = (ws_row(mine.token) * a.num_heads + mine.head) * a.chunk_slots + c;
          if (my_d == 0) {
            a.pmax[slot] = cm;
            static_cast<AccT*>(a.den_ws)[slot] = cd;
          }
          AccT* wp = static_cast<AccT*>(a.wv_ws) + slot * D + my_d;
#pragma unroll
          for (int v = 0; v < VPT; ++v) wp[v] = cw[v];
        } else if (cm != -__builtin_inff()) {
          float Mn, fa, fb;
          merge_factors(M, cm, Mn, fa, fb);
          Dn = wadd<BITS>(rescale<BITS>(Dn, fa), rescale<BITS>(cd, fb));
#pragma unroll
          for (int v = 0; v < VPT; ++v) W[v] = wadd<BITS>(rescale<BITS>(W[v], fa), rescale<BITS>(cw[v], fb));
          M = Mn;
        }
      }
      // (the next chunk's first barrier stands between these reads and the
      // next writes of the stages and of red_d)
      if (!more) break;
      if constexpr (MAXE == 1) next_k();
    }
  }

  if constexpr (!SPLIT) {
    const RowInfo mine = row_of(my_row);
    if (mine.valid) {
      const float den_f = fmaxf(acc_f32<BITS>(Dn, a.fxp_inv), 1.0e-6f);
      T* o = static_cast<T*>(a.o) + mine.token * a.so_t + int64_t(mine.head) * a.so_h + my_d;
#pragma unroll
      for (int v = 0; v < VPT; ++v) o[v] = Io<DT>::store(div_rn(acc_f32<BITS>(W[v], a.fxp_inv), den_f));
    }
  }
}

// MAXE: no request of the launch has more than 4 MAXE rows in a tile (1: decode
// steps of a group of up to 4). Workgroups per CU that the registers are held to:
// with up to 4 rows three, whose loads in flight hide each other's start (two
// dependent round trips: the request's bounds beside the table entries, then K
// and V), else two.
template <int BITS, int D, int MAXE> constexpr int rows16_wgs() {
  return BITS == 64 || D == 256 ? 1 : MAXE == 1 ? 3 : 2;
}

template <int DT, int BITS, int D, bool SPLIT, bool FAST, int MAXE>
__global__ __launch_bounds__(kThreads, (rows16_wgs<BITS, D, MAXE>())) void attn_mx4_rows16_kernel(Mx4Args m) {
  __shared__ __align__(16) Rows16Lds<BITS, D, MAXE> lds;
  const AttnArgs& a = m.a;
  const int lane = threadIdx.x & 63;
  const int slot_x = int(quotient(blockIdx.x, m.by_heads));
  Rows16 w;
  w.g = int(blockIdx.x) - slot_x * a.num_kv_heads;
  w.r = turned(m, slot_x, int(blockIdx.z * gridDim.y + blockIdx.y));
  // the table entries of the first chunk, where it follows from the launch
  // alone, beside the request's bounds
  Pager pg = make_pager(a, w.r, 0);
  int ent = pg.entry_at(32 * (SPLIT ? int(blockIdx.z) : 0) + (lane & 31));
  w.q_start = ((ConstI32)a.qsl)[w.r];
  w.q_len = ((ConstI32)a.qsl)[w.r + 1] - w.q_start;
  w.seq_len = ((ConstI32)a.seq_lens)[w.r];
  w.ctx = w.seq_len - w.q_len;
  w.seq_len = min(w.seq_len, int(a.lmax));  // keys past the table's are not there
  const int rows_total = w.q_len * a.group;
  w.row0 = blockIdx.y * (MAXE == 4 ? QROWS : 4 * MAXE);
  if (w.row0 >= rows_total) return;                        // uniform
  if (a.pq_rows > 0 && rows_total >= a.pq_rows) return;  // attn_mx4_prompt_kernel's request
  if (a.window > 0) {
    const int i_min = int(quotient(uint32_t(w.row0), m.by_group));
    const int c = max(0, w.ctx + i_min - a.window + 1) / (TILE * CT) + (SPLIT ? int(blockIdx.z) : 0);
    ent = pg.entry_at(32 * c + (lane & 31));
  }
  if constexpr (MAXE == 1) {
    rows16_body<DT, BITS, D, SPLIT, FAST, 1>(m, w, lds, ent);
  } else {
    // (a batch of decode steps beside a few short prompts)
    if (rows_total - w.row0 <= 4) rows16_body<DT, BITS, D, SPLIT, FAST, 1>(m, w, lds, ent);
    else rows16_body<DT, BITS, D, SPLIT, FAST, MAXE>(m, w, lds, ent);
  }
}

// ---------------------------------------------------------------------------
// Prompts: RS sets of 16 query rows a wave. A chunk's K tiles are read twice, for the row
// maxima and, alternating with the V tiles, for the weights, as in attn_impl.h's
// prefill kernels. A step is one tile: it lies in one of two LDS tiles while the
// next one is unpacked into the other between the MFMAs; the two after that are
// on their way in registers, packed. Steps alternate between two halves of the
// code, so LDS addresses and registers are fixed (an odd number of first steps is
// padded with one that only moves data). The table entries of a chunk are one
// vector load, its granules' offsets a lane each, kept for two chunks at once: a
// step's addresses are scalar (scalar loads in the loop are waited for together
// with the LDS reads; moving the lanes on at a chunk's end within the loop cost
// 20 moves a step and a wait for the prefetch).
//
// Four prompts of up to 2048 tokens, 32 heads over 8 of 128, bf16: 208 us, 398
// TFLOP/s of the products that the formula has (the K products are made twice).
// Vector instructions are issued in 60 of 100 cycles, MFMAs run in 27, the LDS
// works in 30; two waves per SIMD leave the rest.
//
// LDS rows are padded: a row's 16-byte chunk x is at row * PITCH + (row / 8) *
// OCT + 16 x, so that every read is a constant away from one address. With 64
// bytes of padding four consecutive rows take different quarters of the banks;
// OCT keeps apart the rows 8 k + .. of a K fragment read (16) and of half a
// wave's transposing V read (32).
template <int D> struct PromptLds {
  static constexpr int PITCH = Lds<D>::ROWB + 64;
  static constexpr int KOCT = 16, VOCT = 32;
  static constexpr int TILEB = TILE * PITCH + 8 * VOCT;
};

// SPLIT: the chunks of a row tile are dealt evenly to pq_splits workgroups; the
// first folds its chunks and leaves the folded state as one record, the others
// a record per chunk.
//
// FAST as in the 16-row kernel, and over a softcap too (CAP): the softcap is
// monotone, so the chunk maximum is the capped maximum of the raw scores, and
// only phase 1 computes a score's tanh.
template <int DT, int BITS, int D, bool SPLIT, bool FAST, bool CAP, int RS>
__global__ __launch_bounds__(kPThreads, D == 256 ? 1 : 2) void attn_mx4_prompt_kernel(Mx4Args m) {
  const AttnArgs& a = m.a;
  using TR = Traits<DT>;
  using T = typename TR::T;
  using AccT = typename AccOf<BITS>::T;
  using RL = PromptLds<D>;
  constexpr int QS = D / 32, DBLK = D / 16, ROWS = RS * PQROWS;
  extern __shared__ __align__(16) unsigned char lds[];  // [2] tiles

  const int tid = threadIdx.x, lane = tid & 63, kg = lane >> 4, i16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int r = int(quotient(blockIdx.x, m.by_heads));
  const int g = int(blockIdx.x) - r * a.num_kv_heads;
  int rtile = int(gridDim.y) - 1 - int(blockIdx.y);  // the longest row tiles first
  if (a.pq_blocks == 0) r = turned(m, r, int(blockIdx.z * gridDim.y + blockIdx.y));
  if (a.pq_blocks > 0) {
    r = __builtin_amdgcn_readfirstlane(flat_block(a, a.pq_blocks - 1 - r, rtile, RS == 2 ? 7 : 6));
    rtile = __builtin_amdgcn_readfirstlane(rtile);
    if (r < 0 || rtile < 0) return;  // uniform
  }
  const int q_start = ((ConstI32)a.qsl)[r];
  const int q_len = ((ConstI32)a.qsl)[r + 1] - q_start;
  const int ctx = ((ConstI32)a.seq_lens)[r] - q_len;
  const int seq_len = min(((ConstI32)a.seq_lens)[r], int(a.lmax));  // keys past the table's are not there
  const int rows_total = q_len * a.group;
  const int row0 = rtile * ROWS;
  if (row0 >= rows_total || rows_total < a.pq_rows) return;  // uniform
  const int wrow0 = row0 + 16 * RS * wave;

  const int i_min = int(quotient(uint32_t(row0), m.by_group));
  const int i_max = int(quotient(uint32_t(min(rows_total - 1, row0 + ROWS - 1)), m.by_group));
  const int hi = a.causal ? min(seq_len, ctx + i_max + 1) : seq_len;
  const int lo = a.window > 0 ? max(0, ctx + i_min - a.window + 1) : 0;
  const int t_lo = lo / TILE;
  const int t_hi = hi > lo ? (hi + TILE - 1) / TILE : t_lo;
  const int c_first = t_lo / CT;
  int c_end = t_hi > t_lo ? (t_hi + CT - 1) / CT : c_first;
  if constexpr (SPLIT) c_end = min(c_end, a.chunk_slots);
  const int nch = max(0, c_end - c_first);
  const int split = SPLIT ? blockIdx.z : 0;
  const int per = SPLIT ? (nch + a.pq_splits - 1) / a.pq_splits : nch;
  const int c_lo = c_first + min(nch, split * per);
  const int c_hi = min(c_first + nch, c_lo + per);

  const Pager pager = make_pager(a, r, seq_len);
  const uint32_t ch = uint32_t(g) * m.c_head, sh = uint32_t(g) * m.s_head;

  auto live_lo = [&](int c) { return max(c * CT, t_lo); };
  auto live_hi = [&](int c) { return min(c * CT + CT, t_hi); };

  // The stream of steps. Chunk c with n live tiles from ta has steps0(n) steps of
  // phase 0 (K tile k, past the last the last again) and 2 n of phase 1 (K, V of
  // tile k / 2).
  auto steps0 = [](int n) { return 2 * ((n + 1) >> 1); };
  // Byte offsets and limits (Pager) of the granules of two chunks, a lane each:
  // granule l of chunk c in lane 32 (c % 2) + l.
  uint32_t oc_lo = 0, oc_hi = 0, os_lo = 0, os_hi = 0, lim_c = 0, lim_s = 0;
  auto open_chunk = [&](int c, int ent, bool mine) __attribute__((always_inline)) {
    const int gq = pager.granule(32 * c + (lane & 31));
    const uint64_t oc = pager.offset(gq, ent, m.c_blk, m.c_slot, ch), os = pager.offset(gq, ent, m.s_blk, m.s_slot, sh);
    oc_lo = mine ? uint32_t(oc) : oc_lo;
    oc_hi = mine ? uint32_t(oc >> 32) : oc_hi;
    os_lo = mine ? uint32_t(os) : os_lo;
    os_hi = mine ? uint32_t(os >> 32) : os_hi;
    lim_c = mine ? pager.limit(gq, m.c_slot) + 3 * (D / 8) : lim_c;
    lim_s = mine ? pager.limit(gq, m.s_slot) : lim_s;
  };
  auto entry_of = [&](int c) { return pager.entry_at(pager.granule(32 * c + (lane & 31))); };
  int ent = 0;  // the table entry of the lane's granule of the chunk after the open ones
  // The staging cursor: the next step to load, and the lane of its chunk's first
  // live granule of the wave.
  int fc = c_lo, fphase = 0, fk = 0, fn = 1, fl = 0;
  auto enter = [&]() __attribute__((always_inline)) {
    const int ta = live_lo(fc);
    fn = live_hi(fc) - ta;
    fl = 32 * (fc & 1) + 4 * (ta - CT * fc) + wave;
  };
  auto advance = [&]() __attribute__((always_inline)) {
    ++fk;
    if (fk >= (fphase ? 2 * fn : steps0(fn))) {
      if (fphase && fc + 1 >= c_hi) {
        --fk;  // past the end: the last tile again
      } else {
        fk = 0;
        fc += fphase;
        fphase ^= 1;
        enter();
      }
    }
  };

  // Staging: the wave moves the tile's granule `wave`, lane l row l / 4, units
  // l % 4.
  struct Staged {
    Units<D> u;
    Scales<D> s;
  };
  const int srow = 16 * wave + (lane >> 2);
  const uint32_t c_off = uint32_t(lane >> 2) * m.c_slot + (lane & 3) * (D / 8), s_off = uint32_t(lane >> 2) * m.s_slot;
  auto at_lane = [](uint32_t x, int l) { return uint32_t(__builtin_amdgcn_readlane(int(x), l)); };
  auto fetch = [&](const uint8_t* codes, const uint8_t* scales, int k) __attribute__((always_inline)) {
    const int l = fl + 4 * min(k, fn - 1);
    const uint8_t* cp = codes + ((uint64_t(at_lane(oc_hi, l)) << 32) | at_lane(oc_lo, l));
    const uint8_t* sp = scales + ((uint64_t(at_lane(os_hi, l)) << 32) | at_lane(os_lo, l));
    Staged x;
    x.u = load_units<D>(cp + min(c_off, at_lane(lim_c, l)));
    x.s = load_scales<D>(sp + min(s_off, at_lane(lim_s, l)));
    return x;
  };
  Staged st[2];  // by the step's parity
  auto refill = [&](Staged& x) __attribute__((always_inline)) {
    const bool v = (fphase & fk) != 0;
    x = fetch(v ? m.vc : m.kc, v ? m.vs : m.ks, fk >> fphase);
    advance();
  };
  const unsigned wr_row = srow * RL::PITCH + (lane & 3) * 16;
  const unsigned k_wr = wr_row + (srow >> 3) * RL::KOCT, v_wr = wr_row + (srow >> 3) * RL::VOCT;
  // unit j of a staged tile into LDS at `at`
  auto put = [&](const Staged& x, unsigned at, int j) __attribute__((always_inline)) {
    lds_store16(lds + at + 64 * j, mx4::unpack8<DT>(x.u.w[j], mx4::scale_of<DT>(x.s.w[j / 4], j % 4)));
  };
  if (c_lo < c_hi) {
    const int c = c_lo + ((lane >> 5) ^ (c_lo & 1));
    open_chunk(c, entry_of(c), true);
    ent = entry_of(c_lo + 2);
    enter();
    refill(st[0]);
    refill(st[1]);
  }

  // The lane's query rows, one of each set of 16.
  u32x4 qf[RS][QS];
  int ks[RS], ke[RS], qp[RS];
  float slope[RS];
#pragma unroll
  for (int u = 0; u < RS; ++u) {
    const RowInfo me = row_at(m, g, q_start, q_len, ctx, seq_len, wrow0 + 16 * u + i16);
    const T* qbase = static_cast<const T*>(a.q) + me.token * a.sq_t + int64_t(me.head) * a.sq_h;
#pragma unroll
    for (int j = 0; j < QS; ++j)
      qf[u][j] = me.valid ? *reinterpret_cast<const u32x4*>(qbase + 32 * j + 8 * kg) : u32x4{0u, 0u, 0u, 0u};
    ks[u] = me.valid ? me.kstart : 0x7fffffff;
    ke[u] = me.valid ? me.kend : 0;
    qp[u] = me.qpos;
    slope[u] = !FAST && a.alibi ? a.alibi[me.head] : 0.0f;
  }
  // (worked out again where it is stored: fewer registers over the loop)
  auto row_of = [&](int u) __attribute__((always_inline)) {
    int row = wrow0 + 16 * u;
    asm volatile("" : "+s"(row));
    return row_at(m, g, q_start, q_len, ctx, seq_len, row + i16);
  };
  auto tile_whole = [&](int t) -> bool {
    bool part = false;
#pragma unroll
    for (int u = 0; u < RS; ++u) part |= !(ks[u] <= t * TILE && t * TILE + TILE <= ke[u]);
    return __builtin_amdgcn_ballot_w64(part) == 0;
  };

  // LDS addresses: the score MFMAs' K rows 8 (i16 / 4) + i16 % 4 (h: 4 rows on, s:
  // 32 rows on), chunks 4 j + kg; the transposing V reads, rows 8 kg + i16 / 4,
  // columns 4 (i16 % 4) of d block 0 (d block b: 32 b on).
  const unsigned k_rd = (8 * (i16 >> 2) + (i16 & 3)) * RL::PITCH + (i16 >> 2) * RL::KOCT + kg * 16;
  const unsigned v_rd = (8 * kg + (i16 >> 2)) * RL::PITCH + kg * RL::VOCT + (i16 & 3) * 8;
  constexpr unsigned kStepK = 32 * RL::PITCH + 4 * RL::KOCT, kStepV = 32 * RL::PITCH + 4 * RL::VOCT;

  float Mr[RS];
  AccT Dr[RS];
  AccT Wr[RS][DBLK][4];
#pragma unroll
  for (int u = 0; u < RS; ++u) {
    Mr[u] = -__builtin_inff();
    Dr[u] = 0;
#pragma unroll
    for (int b = 0; b < DBLK; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) Wr[u][b][e] = 0;
  }

  auto store_record = [&](int u, int c, float mc, AccT den, const AccT (&w)[DBLK][4]) __attribute__((always_inline)) {
    const RowInfo me = row_of(u);
    if (!me.valid) return;
    const int64_t slot = (me.token * a.num_heads + me.head) * a.chunk_slots + c;
    if (kg == 0) {
      a.pmax[slot] = mc;
      static_cast<AccT*>(a.den_ws)[slot] = den;
    }
    typedef AccT acc4 __attribute__((ext_vector_type(4)));
    acc4* wp = reinterpret_cast<acc4*>(static_cast<AccT*>(a.wv_ws) + slot * D + 4 * kg);
#pragma unroll
    for (int b = 0; b < DBLK; ++b) wp[4 * b] = acc4{w[b][0], w[b][1], w[b][2], w[b][3]};
  };

  // The four score MFMA chains of a K tile; a chain's LDS reads go out before
  // the chain before it is waited for, and side(q) is done beside chain q.
  auto scores_of = [&](const unsigned char* tile, auto&& side, auto&& fn) __attribute__((always_inline)) {
    u32x4 kf[2][QS];
    auto issue = [&](auto qc) __attribute__((always_inline)) {
      constexpr int q = decltype(qc)::value;
#pragma unroll
      for (int j = 0; j < QS; ++j) kf[q & 1][j] = lds_load16(tile + k_rd + ((q >> 1) * kStepK + (q & 1) * 4 * RL::PITCH + 64 * j));
    };
    issue(std::integral_constant<int, 0>{});
    f32x4 accs[2][RS];
    static_for<4>([&](auto qc) __attribute__((always_inline)) {
      constexpr int q = decltype(qc)::value;
      if constexpr (q + 1 < 4) issue(std::integral_constant<int, q + 1>{});
#pragma unroll
      for (int u = 0; u < RS; ++u) accs[q & 1][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < QS; ++j)
#pragma unroll
        for (int u = 0; u < RS; ++u) accs[q & 1][u] = TR::mma(kf[q & 1][j], qf[u][j], accs[q & 1][u]);
      side(qc);
      if constexpr (q > 0)
#pragma unroll
        for (int u = 0; u < RS; ++u) fn(std::integral_constant<int, q - 1>{}, u, accs[(q - 1) & 1][u]);
      __builtin_amdgcn_sched_barrier(0);
    });
#pragma unroll
    for (int u = 0; u < RS; ++u) fn(std::integral_constant<int, 3>{}, u, accs[1][u]);
  };
  auto capped = [&](float x) { return softcapped(x, a.softcap_log2); };
  // Scores of chain q for the lane's row and keys t * TILE + 32 (q / 2) + 8 kg +
  // 4 (q % 2) + e. (RAW: before the softcap; the mask is -inf, a score is not.)
  auto chain_scores = [&](const f32x4& acc, int t, int u, int q, bool whole, auto raw_tag, float (&sc)[4])
                          __attribute__((always_inline)) {
    constexpr bool RAW = decltype(raw_tag)::value;
    const int key0 = t * TILE + 32 * (q >> 1) + 8 * kg + 4 * (q & 1);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = __fmul_rn(acc[e], a.scale_log2);
      if constexpr (!FAST) {
        if (a.softcap_log2 > 0.0f) x = capped(x);
        if (a.alibi) x = x + slope[u] * static_cast<float>(key0 + e - qp[u]);
      } else if constexpr (CAP) {
        x = RAW ? fmaxf(x, -kFltMax) : capped(x);
      }
      sc[e] = (whole || (key0 + e >= ks[u] && key0 + e < ke[u])) ? x : -__builtin_inff();
    }
  };

  if (c_lo < c_hi) {
    // the first step's tile to LDS; two more on their way
#pragma unroll
    for (int j = 0; j < QS; ++j) put(st[0], k_wr, j);
    refill(st[0]);
    // part q (of four) of unpacking the tile of the step after one of parity P
    constexpr int UPP = QS >= 4 ? QS / 4 : 1;
    auto put_part = [&](auto pc, unsigned at, auto qc) __attribute__((always_inline)) {
      constexpr int P = decltype(pc)::value, q = decltype(qc)::value;
#pragma unroll
      for (int j = q * UPP; j < (q + 1) * UPP && j < QS; ++j) put(st[P ^ 1], (P ^ 1) * RL::TILEB + at, j);
    };

    for (int c = c_lo; c < c_hi; ++c) {
      const int ta = live_lo(c), te = live_hi(c), n0 = steps0(te - ta);
      // (the cursor has left chunk c - 1 and is in chunk c: both have four steps or more)
      if (c > c_lo && c + 1 < c_hi) {
        open_chunk(c + 1, ent, (lane >> 5) == ((c + 1) & 1));
        ent = entry_of(c + 2);
      }
      float mx[RS], mraw[RS];
#pragma unroll
      for (int u = 0; u < RS; ++u) mx[u] = mraw[u] = -__builtin_inff();
      // phase 0: the chunk's row maxima
      auto max_tile = [&](int t, const unsigned char* tile, auto&& side) __attribute__((always_inline)) {
        if (FAST && tile_whole(t)) {
          scores_of(tile, side, [&](auto, int u, const f32x4& acc) __attribute__((always_inline)) {
            mraw[u] = fmaxf(fmaxf(mraw[u], fmaxf(acc[0], acc[1])), fmaxf(acc[2], acc[3]));
          });
          if constexpr (CAP)  // keys were seen
#pragma unroll
            for (int u = 0; u < RS; ++u) mraw[u] = fmaxf(mraw[u], -kFltMax);
        } else {
          scores_of(tile, side, [&](auto qc, int u, const f32x4& acc) __attribute__((always_inline)) {
            float sc[4];
            chain_scores(acc, t, u, decltype(qc)::value, false, std::true_type{}, sc);
            mx[u] = fmaxf(fmaxf(mx[u], fmaxf(sc[0], sc[1])), fmaxf(sc[2], sc[3]));
          });
        }
      };
      auto step0 = [&](auto pc, int t) __attribute__((always_inline)) {
        constexpr int P = decltype(pc)::value;
        lds_barrier();
        if (t < te) max_tile(t, lds + P * RL::TILEB, [&](auto qc) { put_part(pc, k_wr, qc); });
        else static_for<4>([&](auto qc) { put_part(pc, k_wr, qc); });
        refill(st[P ^ 1]);
      };
      for (int k = 0; k < n0; k += 2) {
        step0(std::integral_constant<int, 0>{}, ta + k);
        step0(std::integral_constant<int, 1>{}, ta + k + 1);
      }
      float mrow[RS];
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        if constexpr (FAST) {
          float m1 = __fmul_rn(mraw[u], a.scale_log2);
          if constexpr (CAP) m1 = mraw[u] != -__builtin_inff() ? fmaxf(m1, -kFltMax) : m1;
          mx[u] = fmaxf(mx[u], m1);
        }
        mx[u] = fmaxf(mx[u], __shfl_xor(mx[u], 16, 64));
        mx[u] = fmaxf(mx[u], __shfl_xor(mx[u], 32, 64));
        if constexpr (CAP) mx[u] = mx[u] != -__builtin_inff() ? capped(mx[u]) : mx[u];
        mrow[u] = mx[u] != -__builtin_inff() ? mx[u] : 0.0f;  // no key: pin to 0
      }
      // phase 1: weights and weighted V. FAST: the sums carry kRound per added
      // term, taken out at the chunk's end.
      AccT den[RS];
      AccT wv[RS][DBLK][4];
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        den[u] = 0;
#pragma unroll
        for (int b = 0; b < DBLK; ++b)
#pragma unroll
          for (int e = 0; e < 4; ++e) wv[u][b][e] = 0;
      }
      constexpr std::integral_constant<int, 0> kEven{};
      constexpr std::integral_constant<int, 1> kOdd{};
      for (int t = ta; t < te; ++t) {
        lds_barrier();
        u32x4 pb[RS][2];
        auto weights = [&](auto whole_tag) __attribute__((always_inline)) {
          constexpr bool WHOLE = decltype(whole_tag)::value;
          scores_of(lds, [&](auto qc) { put_part(kEven, v_wr, qc); }, [&](auto qc, int u, const f32x4& acc)
                    __attribute__((always_inline)) {
            constexpr int q = decltype(qc)::value, s = q >> 1, h = q & 1;
            float sc[4], w[4];
            chain_scores(acc, t, u, q, WHOLE, std::false_type{}, sc);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(sc[e] - mrow[u]);
            if constexpr (FAST) {
#pragma unroll
              for (int e = 0; e < 4; ++e)  // (the maximum: NaN counts as 0)
                den[u] = AccT(uint32_t(den[u]) + __float_as_uint(fmaxf(__builtin_fmaf(w[e], a.fxp_scale, kRoundF), kRoundF)));
              pb[u][s][2 * h] = p_pack2<DT>(w[0], w[1]);
              pb[u][s][2 * h + 1] = p_pack2<DT>(w[2], w[3]);
            } else {
              uint32_t p16[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                den[u] = wadd<BITS>(den[u], quant<BITS>(__fmul_rn(w[e], a.fxp_scale)));
                p16[e] = Io<DT>::store(w[e]);
              }
              pb[u][s][2 * h] = p16[0] | (p16[1] << 16);
              pb[u][s][2 * h + 1] = p16[2] | (p16[3] << 16);
            }
          });
        };
        if (FAST && tile_whole(t)) weights(std::true_type{});
        else weights(std::false_type{});
        refill(st[1]);

        // d blocks, the next one's V reads before this one's MFMAs
        lds_barrier();
        const unsigned char* vt = lds + RL::TILEB + v_rd;
        u32x2 vr[2][2][2];
        auto issue_v = [&](auto bc) __attribute__((always_inline)) {
          constexpr int b = decltype(bc)::value;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < 2; ++s) vr[b & 1][s][h] = lds_load_tr8(vt + (s * kStepV + h * 4 * RL::PITCH + 32 * b));
        };
        auto blocks = [&](auto&& fn) __attribute__((always_inline)) {
          issue_v(std::integral_constant<int, 0>{});
          static_for<DBLK>([&](auto bc) __attribute__((always_inline)) {
            constexpr int b = decltype(bc)::value;
            if constexpr (b + 1 < DBLK) issue_v(std::integral_constant<int, b + 1>{});
            f32x4 acc[RS];
#pragma unroll
            for (int u = 0; u < RS; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
              for (int u = 0; u < RS; ++u)
                acc[u] = TR::mma(u32x4{vr[b & 1][s][0][0], vr[b & 1][s][0][1], vr[b & 1][s][1][0], vr[b & 1][s][1][1]},
                                 pb[u][s], acc[u]);
            fn(bc, acc);
            __builtin_amdgcn_sched_barrier(0);
          });
        };
        auto term = [&](float x) { return __float_as_uint(__builtin_fmaf(x, a.fxp_scale, kRoundF)); };
        float vmax = 0.0f;
        f32x4 prev[RS];
        auto add_terms = [&](int b) __attribute__((always_inline)) {
#pragma unroll
          for (int u = 0; u < RS; ++u) {
            vmax = absmax4(vmax, prev[u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) wv[u][b][e] = AccT(uint32_t(wv[u][b][e]) + term(prev[u][e]));
          }
        };
        blocks([&](auto bc, const f32x4 (&acc)[RS]) __attribute__((always_inline)) {
          constexpr int b = decltype(bc)::value;
          if constexpr (b < 4) put_part(kOdd, k_wr, bc);
          if constexpr (FAST) {
            // block b - 1's terms while block b's MFMAs run
            if constexpr (b > 0) add_terms(b - 1);
#pragma unroll
            for (int u = 0; u < RS; ++u) prev[u] = acc[u];
          } else {
#pragma unroll
            for (int u = 0; u < RS; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) wv[u][b][e] = wadd<BITS>(wv[u][b][e], quant<BITS>(__fmul_rn(acc[u][e], a.fxp_scale)));
          }
        });
        refill(st[0]);
        if constexpr (FAST) {
          add_terms(DBLK - 1);
          if (__builtin_amdgcn_ballot_w64(!(vmax < m.vlim)) != 0) {  // uniform: out of the constant's range
            blocks([&](auto bc, const f32x4 (&acc)[RS]) __attribute__((always_inline)) {
              constexpr int b = decltype(bc)::value;
#pragma unroll
              for (int u = 0; u < RS; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const AccT without = AccT(uint32_t(wv[u][b][e]) - term(acc[u][e]));
                  wv[u][b][e] = AccT(uint32_t(wadd<BITS>(without, quant<BITS>(__fmul_rn(acc[u][e], a.fxp_scale)))) + kRound);
                }
            });
          }
        }
      }
#pragma unroll
      for (int u = 0; u < RS; ++u) {
        if constexpr (FAST) {
          const uint32_t terms = uint32_t(te - ta) * kRound;
          den[u] = AccT(uint32_t(den[u]) - 16u * terms);
#pragma unroll
          for (int b = 0; b < DBLK; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) wv[u][b][e] = AccT(uint32_t(wv[u][b][e]) - terms);
        }
        den[u] = wadd<BITS>(den[u], __shfl_xor(den[u], 16, 64));
        den[u] = wadd<BITS>(den[u], __shfl_xor(den[u], 32, 64));
        if (SPLIT && split > 0) {  // uniform
          store_record(u, c, mx[u], den[u], wv[u]);
        } else if (__builtin_amdgcn_ballot_w64(Mr[u] != -__builtin_inff()) == 0) {
          // nothing folded yet in the wave: the chunk's own sums
#pragma unroll
          for (int b = 0; b < DBLK; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) Wr[u][b][e] = wv[u][b][e];
          Dr[u] = den[u];
          Mr[u] = mx[u];
        } else if (mx[u] != -__builtin_inff()) {
          float Mn, fa, fb;
          merge_factors(Mr[u], mx[u], Mn, fa, fb);
          // fa or fb is 1 (unless both maxima are +inf), and rescale(x, 1) = x for
          // 16- and 32-bit sums: one side is rescaled
          const bool one_a = fa == 1.0f;
          if (BITS != 64 && __builtin_amdgcn_ballot_w64(!(one_a || fb == 1.0f)) == 0) {
            const float f = one_a ? fb : fa;
            Dr[u] = wadd<BITS>(rescale<BITS>(one_a ? den[u] : Dr[u], f), one_a ? Dr[u] : den[u]);
#pragma unroll
            for (int b = 0; b < DBLK; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const AccT x = one_a ? wv[u][b][e] : Wr[u][b][e], y = one_a ? Wr[u][b][e] : wv[u][b][e];
                Wr[u][b][e] = wadd<BITS>(rescale<BITS>(x, f), y);
              }
          } else {
            Dr[u] = wadd<BITS>(rescale<BITS>(Dr[u], fa), rescale<BITS>(den[u], fb));
#pragma unroll
            for (int b = 0; b < DBLK; ++b)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                Wr[u][b][e] = wadd<BITS>(rescale<BITS>(Wr[u][b][e], fa), rescale<BITS>(wv[u][b][e], fb));
          }
          Mr[u] = Mn;
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < RS; ++u) {
    const RowInfo me = row_of(u);
    if constexpr (SPLIT) {
      if (split == 0) {
        if (c_lo < c_hi) store_record(u, c_hi - 1, Mr[u], Dr[u], Wr[u]);
        if (me.valid && kg == 0) {
          int* cr = a.crange + 2 * (me.token * a.num_heads + me.head);
          cr[0] = c_lo < c_hi ? c_hi - 1 : c_first;
          cr[1] = c_end;
        }
      }
    } else if (me.valid) {
      // the row's quotients over one denominator by its rounded reciprocal: the
      // bits of div_rn
      const float den_f = fmaxf(acc_f32<BITS>(Dr[u], a.fxp_inv), 1.0e-6f);
      const float rcp = div_rn(1.0f, den_f);
      T* orow = static_cast<T*>(a.o) + me.token * a.so_t + int64_t(me.head) * a.so_h;
#pragma unroll
      for (int b = 0; b < DBLK; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float num = acc_f32<BITS>(Wr[u][b][e], a.fxp_inv);
          orow[b * 16 + 4 * kg + e] = Io<DT>::store(BITS == 64 ? div_rn(num, den_f) : div_rn_by_recip(num, den_f, rcp));
        }
    }
  }
}

// Folds the records of each (token, head) in ascending chunk order and divides.
// The fold's factors do not depend on the sums, so 64 chunks' maxima are scanned
// at once, a lane each; a chunk that raises the running maximum (a few of a
// row's) rescales the sums, the terms of the others are only added, in any
// order. A row's records are loaded a batch ahead of their use.
//
// A wave takes a row, D / 64 elements a lane, or (WIDE, for launches of few rows
// of many chunks) the four waves of a workgroup take 64 elements of a row, each a
// quarter of every block of 64 chunks: a wave leaves its sums up to each chunk
// that raises the maximum, and wave 0 rescales and adds those in order. One
// request over 131072 keys, 32 rows of 256 records: 43 us with a thread folding
// step by step, 21.6 with a wave a row, 19.3 with four of which wave 0 folds up to
// the last raise alone, 10.8 so.
template <int DT, int BITS, int D, bool WIDE>
__global__ __launch_bounds__(256) void attn_mx4_combine_kernel(AttnArgs a) {
  using T = typename Traits<DT>::T;
  using AccT = typename AccOf<BITS>::T;
  constexpr int V = WIDE ? 1 : D / 64, PARTS = WIDE ? D / 64 : 1;
  typedef AccT accv __attribute__((ext_vector_type(V)));
  __shared__ AccT part_w[WIDE ? 68 : 1][64];  // up to chunk l of the block; the waves' last sums
  const int lane = threadIdx.x & 63;
  const int wave = WIDE ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const uint32_t unit =
      WIDE ? blockIdx.x : uint32_t(__builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6)));
  const uint32_t th = unit / PARTS;
  const int d = int(unit % PARTS) * 64 + lane * V;
  const uint32_t wrow = th / uint32_t(a.num_heads);  // (past the last row: past every request)
  const int head = int(th - wrow * uint32_t(a.num_heads));
  int64_t token = wrow;
  if (a.tok_cap > 0) {
    const uint32_t r = wrow / uint32_t(a.tok_cap);
    if (r >= uint32_t(a.num_requests)) return;
    const int i = int(wrow - r * uint32_t(a.tok_cap)), q0 = ((ConstI32)a.qsl)[r], q_len = ((ConstI32)a.qsl)[r + 1] - q0;
    if (i >= q_len || (a.pq_rows > 0 && q_len * a.group >= a.pq_rows)) return;
    token = q0 + i;
    if (token < 0 || token >= a.num_tokens) return;
  } else {
    // tokens outside query_start_loc's range belong to no request and are left
    // as they are
    const int64_t used = min<int64_t>(a.num_tokens, ((ConstI32)a.qsl)[a.num_requests]);
    if (token < ((ConstI32)a.qsl)[0] || token >= used) return;
  }
  const float* pm_p = a.pmax + int64_t(th) * a.chunk_slots;
  const AccT* den_p = static_cast<const AccT*>(a.den_ws) + int64_t(th) * a.chunk_slots;
  const AccT* wv_p = static_cast<const AccT*>(a.wv_ws) + int64_t(th) * a.chunk_slots * D + d;
  const int c0 = max(0, __builtin_amdgcn_readfirstlane(a.crange[2 * int64_t(th)]));
  const int c1 = min(a.chunk_slots, __builtin_amdgcn_readfirstlane(a.crange[2 * int64_t(th) + 1]));
  float M = -__builtin_inff();
  AccT Dn = 0, W[V];  // (Dn: wave 0's)
#pragma unroll
  for (int v = 0; v < V; ++v) W[v] = 0;
  constexpr int NB = 16, NH = 64 / NB;
  accv wc[2][NB];
  auto load = [&](int cb, accv (&w)[NB]) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < NB; ++k) w[k] = *reinterpret_cast<const accv*>(wv_p + int64_t(min(cb + k, c1 - 1)) * D);
  };
  float mn = -__builtin_inff();  // the lane's record of the next block
  AccT dn = 0;
  auto load_lane = [&](int cb) __attribute__((always_inline)) {
    const int cl = min(cb + lane, c1 - 1);
    mn = pm_p[cl];
    dn = den_p[cl];
  };
  if (c0 < c1) {
    load(c0 + wave * (WIDE ? NB : 0), wc[0]);
    load_lane(c0);
  }
  for (int cs = c0; cs < c1; cs += 64) {
    // this lane's chunk: its maximum, and the factors of its fold
    const float mc = cs + lane < c1 ? mn : -__builtin_inff();
    const AccT dc = dn;
    if (cs + 64 < c1) load_lane(cs + 64);
    float incl = mc;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const float x = __shfl_up(incl, o, 64);
      if (lane >= o) incl = fmaxf(incl, x);
    }
    float before = __shfl_up(incl, 1, 64);
    before = lane == 0 ? M : fmaxf(M, before);
    float Mn, fa, fb;
    merge_factors(before, mc, Mn, fa, fb);
    const AccT dr = rescale<BITS>(dc, fb);
    const uint64_t seen = __builtin_amdgcn_ballot_w64(mc != -__builtin_inff());
    // (rescale(x, 1) = x for 16- and 32-bit sums)
    const uint64_t moves = BITS == 64 ? seen : seen & __builtin_amdgcn_ballot_w64(fa != 1.0f);
    M = __shfl(fmaxf(before, incl), 63, 64);
    auto term = [&](int l, const accv& w) __attribute__((always_inline)) {
      const float f = __uint_as_float(uint32_t(__builtin_amdgcn_readlane(int(__float_as_uint(fb)), l)));
#pragma unroll
      for (int v = 0; v < V; ++v) W[v] = wadd<BITS>(W[v], rescale<BITS>(w[v], f));
    };
    auto den_term = [&](int l) -> AccT {
      if constexpr (BITS == 64) {
        const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(dr)), l));
        const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(uint64_t(dr) >> 32)), l));
        return AccT((uint64_t(hi) << 32) | lo);
      } else {
        return AccT(__builtin_amdgcn_readlane(int(dr), l));
      }
    };
    // chunks k0 .. of the block in order
    auto fold = [&](int k0, const accv (&w)[NB]) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const int l = k0 + k;  // uniform
        if (!((seen >> l) & 1)) continue;
        if ((moves >> l) & 1) {
          const float g = __uint_as_float(uint32_t(__builtin_amdgcn_readlane(int(__float_as_uint(fa)), l)));
#pragma unroll
          for (int v = 0; v < V; ++v) W[v] = rescale<BITS>(W[v], g);
          Dn = rescale<BITS>(Dn, g);
        }
        term(l, w[k]);
        Dn = wadd<BITS>(Dn, den_term(l));
      }
    };
    if constexpr (WIDE) {
      // the wave's quarter: a sum per run of chunks between those that move
      auto quarter = [&](const accv (&w)[NB]) __attribute__((always_inline)) {
        AccT sum = 0;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          const int l = wave * NB + k;  // uniform
          if ((moves >> l) & 1) {
            part_w[l][lane] = sum;
            sum = 0;
          }
          const float f = __uint_as_float(uint32_t(__builtin_amdgcn_readlane(int(__float_as_uint(fb)), l)));
          if ((seen >> l) & 1) sum = wadd<BITS>(sum, rescale<BITS>(w[k][0], f));
        }
        part_w[64 + wave][lane] = sum;
      };
      if ((cs - c0) & 64) {
        if (cs + 64 < c1) load(cs + 64 + wave * NB, wc[0]);
        quarter(wc[1]);
      } else {
        if (cs + 64 < c1) load(cs + 64 + wave * NB, wc[1]);
        quarter(wc[0]);
      }
      __syncthreads();
      if (wave == 0) {
        // the denominators' sums up to the lane's chunk, its own included
        AccT sum = (seen >> lane) & 1 ? dr : AccT(0);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const AccT x = __shfl_up(sum, o, 64);
          if (lane >= o) sum = wadd<BITS>(sum, x);
        }
        auto minus = [](AccT x, AccT y) { return AccT(uint64_t(x) - uint64_t(y)); };
        AccT done = 0;
        int q = 0;  // the quarter whose sums are being added
        for (uint64_t todo = moves; todo; todo &= todo - 1) {
          const int l = __builtin_ctzll(todo);
          for (; q < l / NB; ++q) W[0] = wadd<BITS>(W[0], part_w[64 + q][lane]);
          const float g = __shfl(fa, l, 64);
          W[0] = rescale<BITS>(wadd<BITS>(W[0], part_w[l][lane]), g);
          const AccT upto = l > 0 ? __shfl(sum, l - 1, 64) : AccT(0);
          Dn = rescale<BITS>(wadd<BITS>(Dn, minus(upto, done)), g);
          done = upto;
        }
        for (; q < 4; ++q) W[0] = wadd<BITS>(W[0], part_w[64 + q][lane]);
        Dn = wadd<BITS>(Dn, minus(__shfl(sum, 63, 64), done));
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        if (cs + h * NB >= c1) break;  // uniform
        if (cs + (h + 1) * NB < c1) load(cs + (h + 1) * NB, wc[(h + 1) & 1]);
        fold(h * NB, wc[h & 1]);
      }
    }
  }
  if (wave != 0) return;
  const float den_f = fmaxf(acc_f32<BITS>(Dn, a.fxp_inv), 1.0e-6f);
  T* o = static_cast<T*>(a.o) + token * a.so_t + int64_t(head) * a.so_h + d;
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = Io<DT>::store(div_rn(acc_f32<BITS>(W[v], a.fxp_inv), den_f));
}

// Waves of a combine launch from which each takes a row, and chunks per row up
// to which one does: below and above, four waves share 64 elements (WIDE).
constexpr int64_t kWideRows = 2048;
constexpr int kWideChunks = 32;

// ---------------------------------------------------------------------------
// Launches.

// Whether the FAST forms serve a launch (the 16-row one without a softcap).
template <int BITS> bool fast_of(const AttnArgs& a) {
  return BITS != 64 && a.fxp_scale <= (BITS == 16 ? 16384.0f : 4194304.0f) && !a.alibi && a.scale_log2 > 0.0f;
}

template <int DT, int BITS, int D, int RS, bool SPLIT, bool FAST, bool CAP>
int launch_prompt(const Mx4Args& m, dim3 grid, hipStream_t st) {
  auto kern = attn_mx4_prompt_kernel<DT, BITS, D, SPLIT, FAST, CAP, RS>;
  constexpr int lds = 2 * PromptLds<D>::TILEB;
  if constexpr (lds > 64 * 1024) {
    static bool done[64] = {};  // by device (benign race: the attribute is idempotent)
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return int(e);
    if (dev >= 64 || !done[dev]) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (e != hipSuccess) return int(e);
      if (dev < 64) done[dev] = true;
    }
  }
  kern<<<grid, kPThreads, lds, st>>>(m);
  return 0;
}

template <int DT, int BITS, int D, int RS, bool SPLIT> int launch_prompt(const Mx4Args& m, dim3 grid, hipStream_t st) {
  if constexpr (BITS != 64) {
    if (fast_of<BITS>(m.a))
      return m.a.softcap_log2 > 0.0f ? launch_prompt<DT, BITS, D, RS, SPLIT, true, true>(m, grid, st)
                                     : launch_prompt<DT, BITS, D, RS, SPLIT, true, false>(m, grid, st);
  }
  return launch_prompt<DT, BITS, D, RS, SPLIT, false, false>(m, grid, st);
}

template <int DT, int BITS, int D> int launch_prompt(const Mx4Args& m, dim3 grid, bool split, int sets, hipStream_t st) {
  if constexpr (row_sets(BITS, D) == 2) {
    if (sets == 2) return split ? launch_prompt<DT, BITS, D, 2, true>(m, grid, st) : launch_prompt<DT, BITS, D, 2, false>(m, grid, st);
  }
  return split ? launch_prompt<DT, BITS, D, 1, true>(m, grid, st) : launch_prompt<DT, BITS, D, 1, false>(m, grid, st);
}

template <int DT, int BITS, int D, bool SPLIT, int MAXE> void launch_rows16(const Mx4Args& m, dim3 grid, hipStream_t st) {
  if constexpr (BITS != 64) {
    if (fast_of<BITS>(m.a) && !(m.a.softcap_log2 > 0.0f)) {
      attn_mx4_rows16_kernel<DT, BITS, D, SPLIT, true, MAXE><<<grid, kThreads, 0, st>>>(m);
      return;
    }
  }
  attn_mx4_rows16_kernel<DT, BITS, D, SPLIT, false, MAXE><<<grid, kThreads, 0, st>>>(m);
}
template <int DT, int BITS, int D> void launch_rows16(const Mx4Args& m, dim3 grid, bool split, int max_e, hipStream_t st) {
  if (max_e == 1) split ? launch_rows16<DT, BITS, D, true, 1>(m, grid, st) : launch_rows16<DT, BITS, D, false, 1>(m, grid, st);
  else if (max_e == 2) split ? launch_rows16<DT, BITS, D, true, 2>(m, grid, st) : launch_rows16<DT, BITS, D, false, 2>(m, grid, st);
  else split ? launch_rows16<DT, BITS, D, true, 4>(m, grid, st) : launch_rows16<DT, BITS, D, false, 4>(m, grid, st);
}

template <int DT, int BITS, int D>
int launch_mx4(Mx4Args m, const Mx4Plan& p, int num_requests, int max_query_len, int64_t num_tokens, hipStream_t st) {
  AttnArgs& a = m.a;
  a.num_splits = p.splits;
  a.pq_splits = p.pq_splits;
  a.tok_cap = p.tok_cap;
  const int64_t max_rows = int64_t(max_query_len > 1 ? max_query_len : 1) * a.group;
  const bool split = p.splits > 1 || p.pq_splits > 1;
  int64_t qtiles = cdiv(max_rows, QROWS);
  if (p.prompt) {
    a.pq_rows = kPrefillRows;
    qtiles = std::min<int64_t>(qtiles, kShortTiles);
    const int64_t rows = int64_t(p.sets) * PQROWS, ptiles = cdiv(max_rows, rows);
    // a flat grid over the tokens where requests x the longest one's tiles
    // would be mostly empty
    const int64_t flat = num_tokens * a.group / rows + num_requests;
    dim3 grid(unsigned(num_requests * a.num_kv_heads), unsigned(ptiles), unsigned(p.pq_splits));
    if (ptiles > 65535 || (num_requests * ptiles - flat) * a.num_kv_heads * p.pq_splits > kFlatEmpty) {
      a.pq_blocks = int(flat);
      grid = dim3(unsigned(flat * a.num_kv_heads), 1, unsigned(p.pq_splits));
    }
    const int e = launch_prompt<DT, BITS, D>(m, grid, p.pq_splits > 1, p.sets, st);
    if (e) return e;
  }
  const dim3 grid(unsigned(num_requests * a.num_kv_heads), unsigned(qtiles), unsigned(p.splits));
  // (rows of the longest request that these workgroups can get)
  const int64_t short_rows = p.prompt ? kPrefillRows - 1 : max_rows;
  launch_rows16<DT, BITS, D>(m, grid, split, short_rows <= 4 ? 1 : short_rows <= 8 ? 2 : 4, st);
  if (!split) return launch_status();
  const int64_t ws_rows = a.tok_cap > 0 ? int64_t(num_requests) * a.tok_cap : num_tokens;
  const int64_t rows = ws_rows * a.num_heads;
  if (rows < kWideRows && a.chunk_slots > kWideChunks)
    attn_mx4_combine_kernel<DT, BITS, D, true><<<dim3(unsigned(rows * (D / 64))), 256, 0, st>>>(a);
  else
    attn_mx4_combine_kernel<DT, BITS, D, false><<<dim3(unsigned(cdiv(rows, 4))), 256, 0, st>>>(a);
  return launch_status();
}

template <int DT, int BITS>
int dispatch_d(const Mx4Args& m, const Mx4Plan& p, int num_requests, int max_query_len, int64_t num_tokens, hipStream_t st) {
  switch (m.a.head_dim) {
    case 64: return launch_mx4<DT, BITS, 64>(m, p, num_requests, max_query_len, num_tokens, st);
    case 128: return launch_mx4<DT, BITS, 128>(m, p, num_requests, max_query_len, num_tokens, st);
    default: return launch_mx4<DT, BITS, 256>(m, p, num_requests, max_query_len, num_tokens, st);
  }
}

int run_mx4_bf16(const Mx4Args& m, const Mx4Plan& p, int bits, int num_requests, int max_query_len, int64_t num_tokens,
                 hipStream_t st);
int run_mx4_f16(const Mx4Args& m, const Mx4Plan& p, int bits, int num_requests, int max_query_len, int64_t num_tokens,
                hipStream_t st);

}  // namespace m4
}  // namespace attn
}  // namespace fxpr
