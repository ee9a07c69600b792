// The paged KV cache in 4 bits (format: mx4.h): the quantising write that
// precedes attention in a step, and the read back of cached tokens.
//
// Both take four lanes a row (one token, kv head and K or V): lane kg holds
// the chunks 4 j + kg, so a block's 32 elements lie in the four lanes (its
// largest magnitude takes two lane exchanges), a 16-bit row's loads and stores
// cover whole 64-byte runs, and the lane's codes are one run of bytes of the
// cache row. Streaming kernels: 2 D bytes of a 16-bit row on one side,
// D / 2 + D / 32 on the other.
#include "fxpr_internal.h"
#include "mx4.h"

namespace fxpr {
namespace {

using mx4::u32x2;
using mx4::u32x4;

struct Mx4CacheArgs {
  char* key;    // rows of the op's own tensors, read by the write, written by the read back
  char* value;
  uint8_t* codes;
  uint8_t* scales;
  const int64_t* slots;
  uint32_t rows;  // tokens x kv heads
  uint32_t kv_heads;
  int64_t num_slots;
  int block_size, ps_shift;                  // log2(block_size), or -1
  int64_t st[2], sh[2];                      // bytes: token and head strides of key, value
  int64_t c_blk, c_half, c_slot, c_head;     // bytes: codes
  int64_t s_blk, s_half, s_slot, s_head;     // bytes: scales
};

// The cache row of a slot, as byte offsets into codes and scales.
__device__ __forceinline__ void cache_row(const Mx4CacheArgs& a, int64_t slot, uint32_t head, int half, int64_t& c,
                                          int64_t& s) {
  const int64_t blk = a.ps_shift >= 0 ? slot >> a.ps_shift : slot / a.block_size;
  const int64_t off = slot - blk * a.block_size;
  c = blk * a.c_blk + half * a.c_half + off * a.c_slot + head * a.c_head;
  s = blk * a.s_blk + half * a.s_half + off * a.s_slot + head * a.s_head;
}

// QS bytes / words of a lane, as the widest accesses their alignment allows.
template <int QS> __device__ __forceinline__ void store_units(uint8_t* p, const uint32_t (&u)[QS]) {
  if constexpr (QS == 2) {
    *reinterpret_cast<u32x2*>(p) = u32x2{u[0], u[1]};
  } else {
#pragma unroll
    for (int j = 0; j < QS; j += 4) reinterpret_cast<u32x4*>(p)[j / 4] = u32x4{u[j], u[j + 1], u[j + 2], u[j + 3]};
  }
}
template <int QS> __device__ __forceinline__ void load_units(const uint8_t* p, uint32_t (&u)[QS]) {
  if constexpr (QS == 2) {
    const u32x2 v = *reinterpret_cast<const u32x2*>(p);
    u[0] = v[0];
    u[1] = v[1];
  } else {
#pragma unroll
    for (int j = 0; j < QS; j += 4) {
      const u32x4 v = reinterpret_cast<const u32x4*>(p)[j / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[j + i] = v[i];
    }
  }
}

// Eight elements at p as fp32.
template <int DT> __device__ __forceinline__ void load8(const char* p, float (&x)[8]) {
  if constexpr (DT == FXPR_DTYPE_F32) {
    const u32x4 lo = reinterpret_cast<const u32x4*>(p)[0], hi = reinterpret_cast<const u32x4*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = __uint_as_float(lo[i]);
      x[4 + i] = __uint_as_float(hi[i]);
    }
  } else {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Io<DT>::load(uint16_t(v[i / 2] >> (16 * (i & 1))));
  }
}

// One row per four lanes, K (blockIdx.y 0) or V (1). Each input element is
// read once and each cache byte written once. The arithmetic is exact but for
// the code itself: amax by integer maximum of the magnitudes' bits, a power of
// two as the scale, v_cvt_scalef32_pk_fp4_f32 rounding x / s half to even and
// saturating at 6 (swept against this definition over its whole input range).
template <int DT, int D> __global__ __launch_bounds__(256) void write_mx4_kernel(Mx4CacheArgs a) {
  constexpr int QS = D / 32, ESZ = DT == FXPR_DTYPE_F32 ? 4 : 2;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = min(idx >> 2, a.rows - 1), kg = idx & 3;  // (whole waves: the lane exchanges need them)
  const int half = blockIdx.y;
  const uint32_t t = row / a.kv_heads, h = row - t * a.kv_heads;
  const int64_t slot = a.slots[t];
  const char* src = (half ? a.value : a.key) + int64_t(t) * a.st[half] + int64_t(h) * a.sh[half] + kg * (8 * ESZ);
  float x[QS][8];
#pragma unroll
  for (int j = 0; j < QS; ++j) load8<DT>(src + j * (32 * ESZ), x[j]);
  uint32_t units[QS], bytes[QS];
#pragma unroll
  for (int j = 0; j < QS; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[j][i] = x[j][i] == x[j][i] ? x[j][i] : 0.0f;  // NaN -> 0
      m = max(m, __float_as_uint(x[j][i]) & 0x7fffffffu);
    }
    m = max(m, uint32_t(__shfl_xor(int(m), 1, 64)));
    m = max(m, uint32_t(__shfl_xor(int(m), 2, 64)));
    bytes[j] = mx4::scale_byte<DT>(m);
    const float s = __uint_as_float(bytes[j] << 23);
    uint32_t u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[j][0], x[j][1], s, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[j][2], x[j][3], s, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[j][4], x[j][5], s, 2);
    units[j] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, x[j][6], x[j][7], s, 3);
  }
  if (idx >> 2 >= a.rows || slot < 0 || slot >= a.num_slots) return;
  int64_t c, so;
  cache_row(a, slot, h, half, c, so);
  store_units<QS>(a.codes + c + kg * (QS * 4), units);
  if (kg == 0) {
    uint8_t* sp = a.scales + so;
    if constexpr (QS == 2) {
      *reinterpret_cast<uint16_t*>(sp) = uint16_t(bytes[0] | (bytes[1] << 8));
    } else {
#pragma unroll
      for (int j = 0; j < QS; j += 4)
        reinterpret_cast<uint32_t*>(sp)[j / 4] =
            bytes[j] | (bytes[j + 1] << 8) | (bytes[j + 2] << 16) | (bytes[j + 3] << 24);
    }
  }
}

// The rows of the listed slots as floats, [n, kv heads, D] contiguous; a slot
// outside the cache (padding) gives zeros.
template <int DT, int D> __global__ __launch_bounds__(256) void gather_mx4_kernel(Mx4CacheArgs a) {
  constexpr int QS = D / 32, ESZ = DT == FXPR_DTYPE_F32 ? 4 : 2;
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = idx >> 2, kg = idx & 3;
  if (row >= a.rows) return;
  const int half = blockIdx.y;
  const uint32_t t = row / a.kv_heads, h = row - t * a.kv_heads;
  const int64_t slot = a.slots[t];
  char* dst = (half ? a.value : a.key) + int64_t(row) * (D * ESZ) + kg * (8 * ESZ);
  if (slot < 0 || slot >= a.num_slots) {
#pragma unroll
    for (int j = 0; j < QS; ++j)
#pragma unroll
      for (int i = 0; i < ESZ / 2; ++i) *reinterpret_cast<u32x4*>(dst + j * (32 * ESZ) + 16 * i) = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  int64_t c, so;
  cache_row(a, slot, h, half, c, so);
  uint32_t units[QS], sw[(QS + 3) / 4];
  load_units<QS>(a.codes + c + kg * (QS * 4), units);
  if constexpr (QS == 2) {
    sw[0] = *reinterpret_cast<const uint16_t*>(a.scales + so);
  } else {
#pragma unroll
    for (int j = 0; j < QS / 4; ++j) sw[j] = reinterpret_cast<const uint32_t*>(a.scales + so)[j];
  }
#pragma unroll
  for (int j = 0; j < QS; ++j) {
    const float s = mx4::scale_of<DT>(sw[j / 4], j % 4);
    u32x4* p = reinterpret_cast<u32x4*>(dst + j * (32 * ESZ));
    if constexpr (DT == FXPR_DTYPE_F32) {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(units[j], s, 0);
      const f32x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(units[j], s, 1);
      const f32x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(units[j], s, 2);
      const f32x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(units[j], s, 3);
      p[0] = u32x4{__float_as_uint(v0[0]), __float_as_uint(v0[1]), __float_as_uint(v1[0]), __float_as_uint(v1[1])};
      p[1] = u32x4{__float_as_uint(v2[0]), __float_as_uint(v2[1]), __float_as_uint(v3[0]), __float_as_uint(v3[1])};
    } else {
      p[0] = mx4::unpack8<DT>(units[j], s);
    }
  }
}

template <int DT, int D> void launch(bool write, const Mx4CacheArgs& a, hipStream_t st) {
  const dim3 grid(unsigned(cdiv(int64_t(a.rows) * 4, 256)), 2);
  if (write) write_mx4_kernel<DT, D><<<grid, 256, 0, st>>>(a);
  else gather_mx4_kernel<DT, D><<<grid, 256, 0, st>>>(a);
}

template <int DT> void launch_d(bool write, const Mx4CacheArgs& a, int d, hipStream_t st) {
  switch (d) {
    case 64: return launch<DT, 64>(write, a, st);
    case 128: return launch<DT, 128>(write, a, st);
    default: return launch<DT, 256>(write, a, st);
  }
}

int run(bool write, Mx4CacheArgs& a, int dtype, int64_t num_tokens, int num_kv_heads, int head_size, int block_size,
        int64_t num_blocks, const int64_t* strides, void* stream) {
  if (dtype != FXPR_DTYPE_F16 && dtype != FXPR_DTYPE_BF16 && dtype != FXPR_DTYPE_F32) return FXPR_E_DTYPE;
  if (num_tokens < 0 || num_kv_heads <= 0 || block_size <= 0 || num_blocks < 0) return FXPR_E_SHAPE;
  if (head_size != 64 && head_size != 128 && head_size != 256) return FXPR_E_SHAPE;
  if (num_tokens == 0 || (write && num_blocks == 0)) return FXPR_OK;
  if (!a.key || !a.value || !a.slots || (num_blocks > 0 && (!a.codes || !a.scales))) return FXPR_E_ARG;
  if (num_tokens > (int64_t(1) << 30) / num_kv_heads) return FXPR_E_SHAPE;  // (four 32-bit thread indices a row)
  // 16-byte loads of the codes (a row's D / 2 bytes are whole ones) and of the
  // float rows, D / 32 bytes of scales at once
  const int sb = head_size / 32;
  for (int i = 0; i < 4; ++i)
    if (strides[i] % 16 != 0 || strides[4 + i] % sb != 0) return FXPR_E_ARG;
  if (!aligned(a.codes, 16) || !aligned(a.scales, uintptr_t(sb)) || !aligned(a.key, 16) || !aligned(a.value, 16))
    return FXPR_E_ARG;
  a.rows = uint32_t(num_tokens * num_kv_heads);
  a.kv_heads = uint32_t(num_kv_heads);
  a.num_slots = num_blocks * block_size;
  a.block_size = block_size;
  a.ps_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(unsigned(block_size)) : -1;
  a.c_blk = strides[0];
  a.c_half = strides[1];
  a.c_slot = strides[2];
  a.c_head = strides[3];
  a.s_blk = strides[4];
  a.s_half = strides[5];
  a.s_slot = strides[6];
  a.s_head = strides[7];
  hipStream_t st = as_stream(stream);
  switch (dtype) {
    case FXPR_DTYPE_F16: launch_d<FXPR_DTYPE_F16>(write, a, head_size, st); break;
    case FXPR_DTYPE_BF16: launch_d<FXPR_DTYPE_BF16>(write, a, head_size, st); break;
    default: launch_d<FXPR_DTYPE_F32>(write, a, head_size, st); break;
  }
  return launch_status();
}

}  // namespace
}  // namespace fxpr

using namespace fxpr;

extern "C" int fxpr_reshape_and_cache_mx4(const void* key, const void* value, void* codes, void* scales, int dtype,
                                          const int64_t* slot_mapping, int64_t num_tokens, int num_kv_heads,
                                          int head_size, int block_size, int64_t num_blocks, int64_t stride_key_token,
                                          int64_t stride_key_head, int64_t stride_value_token, int64_t stride_value_head,
                                          int64_t stride_codes_block, int64_t stride_codes_half,
                                          int64_t stride_codes_slot, int64_t stride_codes_head,
                                          int64_t stride_scales_block, int64_t stride_scales_half,
                                          int64_t stride_scales_slot, int64_t stride_scales_head, void* stream) {
  const int esz = dtype == FXPR_DTYPE_F32 ? 4 : 2;
  Mx4CacheArgs a{};
  a.key = const_cast<char*>(static_cast<const char*>(key));
  a.value = const_cast<char*>(static_cast<const char*>(value));
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(scales);
  a.slots = slot_mapping;
  a.st[0] = stride_key_token * esz;
  a.sh[0] = stride_key_head * esz;
  a.st[1] = stride_value_token * esz;
  a.sh[1] = stride_value_head * esz;
  for (int64_t s : {a.st[0], a.sh[0], a.st[1], a.sh[1]})
    if (s % 16 != 0 && num_tokens > 0) return FXPR_E_ARG;
  const int64_t strides[] = {stride_codes_block,  stride_codes_half,  stride_codes_slot,  stride_codes_head,
                             stride_scales_block, stride_scales_half, stride_scales_slot, stride_scales_head};
  return run(true, a, dtype, num_tokens, num_kv_heads, head_size, block_size, num_blocks, strides, stream);
}

extern "C" int fxpr_gather_cache_mx4(const void* codes, const void* scales, void* key, void* value, int dtype,
                                     const int64_t* slot_mapping, int64_t num_slots, int num_kv_heads, int head_size,
                                     int block_size, int64_t num_blocks, int64_t stride_codes_block,
                                     int64_t stride_codes_half, int64_t stride_codes_slot, int64_t stride_codes_head,
                                     int64_t stride_scales_block, int64_t stride_scales_half,
                                     int64_t stride_scales_slot, int64_t stride_scales_head, void* stream) {
  Mx4CacheArgs a{};
  a.key = static_cast<char*>(key);
  a.value = static_cast<char*>(value);
  a.codes = const_cast<uint8_t*>(static_cast<const uint8_t*>(codes));
  a.scales = const_cast<uint8_t*>(static_cast<const uint8_t*>(scales));
  a.slots = slot_mapping;
  const int64_t strides[] = {stride_codes_block,  stride_codes_half,  stride_codes_slot,  stride_codes_head,
                             stride_scales_block, stride_scales_half, stride_scales_slot, stride_scales_head};
  return run(false, a, dtype, num_slots, num_kv_heads, head_size, block_size, num_blocks, strides, stream);
}
