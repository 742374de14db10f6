// Rotary positions in their general form fused with the cache write, and the 8-bit (e4m3) cache: its write and its
// read-back. No counterpart in the reference (one rotary form, forgeserve/model.py:34-45; a cache in the model's type).
//
// Rotation of the first `rd` values of a q or k head by the token's (c_i, s_i), i < rd/2 (fp32 tables):
//     (a, b) -> (a c - b s, b c + a s),   (a, b) = (x[i], x[i + rd/2])  half layout
//                                         (a, b) = (x[2i], x[2i + 1])   interleaved layout
// and x[rd..hd) is copied. Arithmetic is fp32 with one rounding at the end: these forms have no bf16 reference whose
// intermediate roundings would have to be kept (rope_kv_kernel in elementwise.cu keeps them for the plain form).
//
// 8-bit cache: a (slot, KV head) row of hd values has one fp32 scale = max(max|x| / 448, 2^-126) and hd codes
// e4m3(x / scale), rounded to nearest even; 448 is e4m3's largest value, and the floor on the scale keeps 1 / scale
// finite (a row of zeros gets zero codes). A row holding an infinity or a NaN gets an infinite or NaN scale and reads
// back as NaN. A scale for each row costs 4 bytes on hd and needs no calibration, and a row can be written without
// reading its block. Codes lie as the values of an unquantised cache do; scales as (num_blocks, n_kv, block_size).
//
// A negative position marks a padding token: its q_out row and the cache stay as they were.
#include "common.cuh"
#include "kernels.h"
#include "quant.cuh"

namespace fs {

namespace {

struct WriteParams {
  const void* qkv;
  int64_t ld;
  void* q_out;
  int64_t ldq;
  const float* cos_t;
  const float* sin_t;
  int64_t rope_rows;
  int rd;                     // rotated values a head (even, <= hd)
  const int64_t* positions;   // (B, T), contiguous
  KVCache kv;                 // values in the activation type, or e4m3 codes
  KVScales sc;                // quantised cache only
  int T_new, nh, nkv, hd;
  int64_t tokens, slot_base;
  int slot_from_pos;
  unsigned* err;
};

// The cache row of a token: element offset of its values in KV head 0 and of its scale, or -1 where the block table
// does not cover the slot.
struct Slot {
  int64_t values, scale;
};
__device__ __forceinline__ Slot find_slot(const WriteParams& p, int64_t tok, int64_t pos, bool report) {
  const int64_t r = tok / p.T_new;
  const int64_t slot = p.slot_from_pos ? pos : p.slot_base + (tok - r * p.T_new);
  int64_t col, in;
  split_slot(slot, p.kv.block_size, col, in);
  int64_t blk = -1;
  if (col < p.kv.table_cols) blk = p.kv.table[r * p.kv.table_stride + col];
  if (blk < 0 || blk >= p.kv.num_blocks) {
    if (report) flag_error(p.err, ERR_BAD_SLOT);
    return {-1, -1};
  }
  return {blk * p.kv.block_stride + in * p.hd, blk * p.sc.block_stride + in};
}

// Whether the token is real and its position lies in the tables; flags a position past them.
__device__ __forceinline__ bool token_ok(const WriteParams& p, int64_t pos, bool report) {
  if (pos < 0) return false;
  if (p.rd > 0 && pos >= p.rope_rows) {
    if (report) flag_error(p.err, ERR_BAD_POSITION);
    return false;
  }
  return true;
}

// One warp a (token, head), any even hd up to 512 and any alignment. A lane owns whole pairs (the rotated ones, then
// neighbours of the copied rest), so a head may be rewritten in place.
template <typename T, bool QUANT>
__global__ void __launch_bounds__(256) rotary_write_kernel(WriteParams p, int interleaved) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  constexpr int MAXP = 8;   // pairs a lane: hd / 64
  const int lane = threadIdx.x & 31, heads = p.nh + 2 * p.nkv;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int64_t tok = item / heads;
  const int h = static_cast<int>(item - tok * heads);
  if (tok >= p.tokens) return;   // whole warps leave
  const int64_t pos = p.positions[tok];
  const bool report = h == 0 && lane == 0;
  if (!token_ok(p, pos, report)) return;
  const bool turns = h < p.nh + p.nkv;
  const int half = p.rd / 2, pairs = p.hd / 2;
  const T* x = static_cast<const T*>(p.qkv) + tok * p.ld + static_cast<int64_t>(h) * p.hd;
  float a[MAXP], b[MAXP];
  int ia[MAXP], ib[MAXP];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < MAXP; ++j) {
    const int i = lane + 32 * j;
    if (i >= pairs) break;
    const bool rot = turns && i < half;
    ia[j] = rot && !interleaved ? i : (turns && !interleaved ? p.rd + 2 * (i - half) : 2 * i);
    ib[j] = rot && !interleaved ? i + half : ia[j] + 1;
    a[j] = to_f(x[ia[j]]);
    b[j] = to_f(x[ib[j]]);
    if (rot) {
      const float c = p.cos_t[pos * half + i], s = p.sin_t[pos * half + i];
      const float u = a[j], w = b[j];
      a[j] = u * c - w * s;
      b[j] = w * c + u * s;
    }
    top = max(top, max(abs_bits(a[j]), abs_bits(b[j])));
  }
  if (h < p.nh) {
    T* o = static_cast<T*>(p.q_out) + tok * p.ldq + static_cast<int64_t>(h) * p.hd;
#pragma unroll
    for (int j = 0; j < MAXP; ++j) {
      if (lane + 32 * j >= pairs) break;
      o[ia[j]] = from_f<T>(a[j]);
      o[ib[j]] = from_f<T>(b[j]);
    }
    if (p.nkv > 0 && h == 0) find_slot(p, tok, pos, report);   // only to report a bad slot once a token
    return;
  }
  const Slot at = find_slot(p, tok, pos, p.nh == 0 && report);
  if (at.values < 0) return;
  const bool is_v = h >= p.nh + p.nkv;
  const int g = h - p.nh - (is_v ? p.nkv : 0);
  if constexpr (QUANT) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float scale = row_scale(top), inv = 1.f / scale;
    uint8_t* o = static_cast<uint8_t*>(is_v ? p.kv.v : p.kv.k) + at.values + static_cast<int64_t>(g) * p.kv.head_stride;
#pragma unroll
    for (int j = 0; j < MAXP; ++j) {
      if (lane + 32 * j >= pairs) break;
      const uint32_t e = e4m3x2(a[j] * inv, b[j] * inv);
      o[ia[j]] = static_cast<uint8_t>(e);
      o[ib[j]] = static_cast<uint8_t>(e >> 8);
    }
    if (lane == 0) (is_v ? p.sc.v : p.sc.k)[at.scale + static_cast<int64_t>(g) * p.sc.head_stride] = scale;
  } else {
    T* o = static_cast<T*>(is_v ? p.kv.v : p.kv.k) + at.values + static_cast<int64_t>(g) * p.kv.head_stride;
#pragma unroll
    for (int j = 0; j < MAXP; ++j) {
      if (lane + 32 * j >= pairs) break;
      o[ia[j]] = from_f<T>(a[j]);
      o[ib[j]] = from_f<T>(b[j]);
    }
  }
}

// Values of `n_slots` slots of every row, k and v: one thread a value of each.
template <typename T>
__global__ void __launch_bounds__(256)
    kv_dequant_kernel(KVCache kv, KVScales sc, uint32_t n_slots, int nkv, int hd, T* __restrict__ k_out,
                      T* __restrict__ v_out, unsigned* err) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  const int64_t r = blockIdx.z, g = blockIdx.y;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t s = i / hd;
  const int d = static_cast<int>(i - s * hd);
  if (s >= n_slots) return;
  int64_t col, in;
  split_slot(s, kv.block_size, col, in);
  const int64_t blk = col < kv.table_cols ? kv.table[r * kv.table_stride + col] : -1;
  float k = 0.f, v = 0.f;
  if (blk >= 0 && blk < kv.num_blocks) {
    const int64_t at = blk * kv.block_stride + g * kv.head_stride + in * hd + d;
    const int64_t sat = blk * sc.block_stride + g * sc.head_stride + in;
    k = e4m3_to_f(static_cast<const uint8_t*>(kv.k)[at]) * sc.k[sat];
    v = e4m3_to_f(static_cast<const uint8_t*>(kv.v)[at]) * sc.v[sat];
  } else if (d == 0 && in == 0) {
    flag_error(err, ERR_BAD_SLOT);
  }
  const int64_t o = ((r * nkv + g) * n_slots + s) * hd + d;
  k_out[o] = from_f<T>(k);
  v_out[o] = from_f<T>(v);
}

template <typename T>
int write_t(const WriteParams& p, bool quant, int interleaved, cudaStream_t st) {
  const int64_t warps = p.tokens * (p.nh + 2 * p.nkv), blocks = (warps + 7) / 8;
  if (blocks > INT32_MAX) return fail("rotary_kv_write: too many tokens");
  if (quant)
    launch_pdl_async(rotary_write_kernel<T, true>, static_cast<unsigned>(blocks), 256, 0, st, p, interleaved);
  else
    launch_pdl_async(rotary_write_kernel<T, false>, static_cast<unsigned>(blocks), 256, 0, st, p, interleaved);
  return check_launch("rotary_write_kernel");
}

}  // namespace

int rotary_kv_write(int dtype, const void* qkv, int64_t ld, void* q_out, int64_t ldq, const float* cos_t,
                    const float* sin_t, int64_t rope_rows, int64_t rd, int interleaved, const int64_t* positions,
                    const KVCache& kv, const KVScales* sc, int64_t B, int64_t T_new, int64_t nh, int64_t nkv,
                    int64_t hd, int64_t slot_base, int slot_from_pos, cudaStream_t st) {
  WriteParams p;
  p.qkv = qkv;
  p.ld = ld;
  p.q_out = q_out;
  p.ldq = ldq;
  p.cos_t = cos_t;
  p.sin_t = sin_t;
  p.rope_rows = rope_rows;
  p.rd = static_cast<int>(rd);
  p.positions = positions;
  p.kv = kv;
  p.sc = sc ? *sc : KVScales{nullptr, nullptr, 0, 0};
  p.T_new = static_cast<int>(T_new);
  p.nh = static_cast<int>(nh);
  p.nkv = static_cast<int>(nkv);
  p.hd = static_cast<int>(hd);
  p.tokens = B * T_new;
  p.slot_base = slot_base;
  p.slot_from_pos = slot_from_pos;
  p.err = error_word();
  if (!p.err) return -1;
  return dtype == F32 ? write_t<float>(p, sc != nullptr, interleaved, st)
                      : write_t<__nv_bfloat16>(p, sc != nullptr, interleaved, st);
}

int kv_dequant(int dtype, const KVCache& kv, const KVScales& sc, int64_t B, int64_t n_slots, int64_t nkv, int64_t hd,
               void* k_out, void* v_out, cudaStream_t st) {
  unsigned* err = error_word();
  if (!err) return -1;
  const dim3 grid(static_cast<unsigned>((n_slots * hd + 255) / 256), static_cast<unsigned>(nkv),
                  static_cast<unsigned>(B));
  if (dtype == F32)
    launch_pdl_async(kv_dequant_kernel<float>, grid, 256, 0, st, kv, sc, static_cast<uint32_t>(n_slots),
                     static_cast<int>(nkv), static_cast<int>(hd), static_cast<float*>(k_out),
                     static_cast<float*>(v_out), err);
  else
    launch_pdl_async(kv_dequant_kernel<__nv_bfloat16>, grid, 256, 0, st, kv, sc, static_cast<uint32_t>(n_slots),
                     static_cast<int>(nkv), static_cast<int>(hd), static_cast<__nv_bfloat16*>(k_out),
                     static_cast<__nv_bfloat16*>(v_out), err);
  return check_launch("kv_dequant_kernel");
}

}  // namespace fs
