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
// e4m3(x r), rounded to nearest even, with r = 1 / scale to 2^-22: the codes of x / scale, but where that lies within 2^-21
// of itself of a border between two codes either one. 448 is e4m3's largest value, and the floor on the scale keeps 1 / scale
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
  const uint32_t r = static_cast<uint32_t>(tok) / static_cast<uint32_t>(p.T_new);   // tokens are below 2^31
  const int64_t slot = p.slot_from_pos ? pos : p.slot_base + (tok - static_cast<int64_t>(r) * p.T_new);
  int64_t col, in;
  split_slot(slot, p.kv.block_size, col, in);
  int64_t blk = -1;
  if (col < p.kv.table_cols) blk = p.kv.table[static_cast<int64_t>(r) * p.kv.table_stride + col];
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

// What the vector form below does not take: one warp a (token, head), any even hd up to 512 and any alignment. A lane
// owns whole pairs (the rotated ones, then neighbours of the copied rest), so a head may be rewritten in place.
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
    const float scale = row_scale(top), inv = inverse(scale);
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

// A 16-byte piece as fp32 values, and back with one rounding.
__device__ __forceinline__ void unpack_piece(uint4 u, float* x, const __nv_bfloat16*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack_piece(uint4 u, float* x, const float*) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_piece(__nv_bfloat16* p, const float* x) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}
__device__ __forceinline__ void store_piece(float* p, const float* x) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
// max(|a|, |b|, |c|), NaN if one of them is.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// N (2, 4 or 8) table values, N-aligned.
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* x) {
  if constexpr (N == 2) {
    *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(x + i) = *reinterpret_cast<const float4*>(p + i);
  }
}
template <int N>
__device__ __forceinline__ void put_floats(float* p, const float* x) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = *reinterpret_cast<const float4*>(x + i);
}
// N (4 or 8) codes, and their values.
template <int N>
__device__ __forceinline__ uint2 load_codes(const uint8_t* p) {
  if constexpr (N == 8) return *reinterpret_cast<const uint2*>(p);
  return make_uint2(*reinterpret_cast<const uint32_t*>(p), 0);
}
template <int N>
__device__ __forceinline__ void decode_piece(uint2 codes, float scale, float* x) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const uint32_t h = e4m3x2_to_half2(static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1))));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x[2 * i] = f.x * scale;
    x[2 * i + 1] = f.y * scale;
  }
}
// The codes of N (4 or 8) values.
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* p, const float* x, float inv) {
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    w[i] = e4m3x2(x[4 * i] * inv, x[4 * i + 1] * inv) | e4m3x2(x[4 * i + 2] * inv, x[4 * i + 3] * inv) << 16;
  if constexpr (N == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(p) = w[0];
}

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {   // to shared memory
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

// The vector forms, for heads of whole 16-byte pieces (write_vec_ok). A thread owns two pieces of VEC values of a head,
// chosen so that the lanes of a head read neighbouring pieces: x[VEC c ..] and x[r/2 + VEC c ..] where they turn as pairs
// (half layout), the same in the copied rest; first and second half of the head otherwise. It does so for HEADS
// neighbouring heads, so that its cos and sin are read once. The lanes of a head (a power of two, some idle where
// hd / (2 VEC) is none) find the largest |x| by shuffles. The position comes first: a padding token's values are not read.
//
// PAIRS says how a value finds the other one of its pair: HALVES, in the thread's other piece (half layout, r a multiple
// of 2 VEC); NEIGHBOURS, in the same piece (interleaved layout); STAGED, anywhere in the head (half layout, any r).
//
// One wave of CTAs stays, and a thread copies its next item's pieces into shared memory while it works on one (8 ragged
// rows of 2048 tokens of 64 + 8 + 8 heads of 128 to the 8-bit cache: 91 us, 96 % of HBM; loads into registers 105, the
// issue slots being 62 % busy while nothing hides a load). Three CTAs an SM hold all in registers; four spill and put
// more streams on HBM (91 -> 95; fp32 55 -> 62 for 8192 tokens of 32 + 8 + 8 heads).
enum Pairs { HALVES, NEIGHBOURS, STAGED };
template <typename T>
constexpr int VALUES = 16 / static_cast<int>(sizeof(T));   // VEC: values of a piece
constexpr int WRITE_HEADS = 2, WRITE_CTAS = 3;             // HEADS; CTAs an SM

// A lane's place in a head: where its pieces lie, of q and k heads and of v heads.
template <typename T, Pairs PAIRS>
struct Lane {
  static constexpr int VEC = VALUES<T>;
  static constexpr bool IL = PAIRS == NEIGHBOURS;
  int c, lanes, half, heads, lo, hi, lo_v, hi_v;
  bool owns, turns, all_turn;
  __device__ __forceinline__ Lane(const WriteParams& p, int n) {
    lanes = n;
    c = threadIdx.x & (lanes - 1);
    half = p.rd / 2;
    heads = p.nh + 2 * p.nkv;
    owns = c * 2 * VEC < p.hd;
    turns = PAIRS != HALVES || c * 2 * VEC < p.rd;   // IL: pair by pair below,
    all_turn = !IL || p.rd == p.hd;                  // unless all do
    lo = lo_v = VEC * c;
    hi = hi_v = p.hd / 2 + VEC * c;
    if constexpr (PAIRS == HALVES) {
      if (turns) {
        hi = half + VEC * c;
      } else {
        lo = p.rd + VEC * c - half;   // c - rd / (2 VEC) pieces into the rest
        hi = lo + (p.hd - p.rd) / 2;
      }
    }
  }
  __device__ __forceinline__ int pair_of(int i) const {
    return IL ? (i < VEC / 2 ? lo / 2 + i : hi / 2 + i - VEC / 2) : VEC * c + i;
  }
  // cos and sin of the thread's VEC pairs. Pairs past the rotated ones are left alone (not turned by 1 and 0: a NaN or an
  // infinity stays in its own value).
  __device__ __forceinline__ void load_turns(const WriteParams& p, bool ok, int64_t pos, float* cs, float* sn) const {
    const float* ct = p.cos_t + pos * half;
    const float* st = p.sin_t + pos * half;
    if constexpr (PAIRS == STAGED) {
      const int active = p.hd / (2 * VEC);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (ok && c + active * i < half) cs[i] = ct[c + active * i], sn[i] = st[c + active * i];
    } else if constexpr (PAIRS == HALVES) {
      if (ok && turns) {
        load_floats<VEC>(ct + VEC * c, cs);
        load_floats<VEC>(st + VEC * c, sn);
      }
    } else if (ok && half % (VEC / 2) == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += VEC / 2) {
        if (pair_of(i) < half) {
          load_floats<VEC / 2>(ct + pair_of(i), cs + i);
          load_floats<VEC / 2>(st + pair_of(i), sn + i);
        }
      }
    } else if (ok) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (pair_of(i) < half) cs[i] = ct[pair_of(i)], sn[i] = st[pair_of(i)];
    }
  }
  // The lane's pairs of a q or k head.
  __device__ __forceinline__ void turn(float* x, const float* cs, const float* sn) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float& a = x[IL ? 2 * i : i];
      float& b = x[IL ? 2 * i + 1 : VEC + i];
      const float a0 = a, b0 = b;
      if (!IL || all_turn || pair_of(i) < half) {
        a = a0 * cs[i] - b0 * sn[i];
        b = b0 * cs[i] + a0 * sn[i];
      }
    }
  }
  // Stores the lane's values of head h: q to q_row, k and v to the cache. mine: the head is the lane's; all lanes call.
  template <bool QUANT>
  __device__ __forceinline__ void put(const WriteParams& p, bool mine, int h, const float* x, T* q_row,
                                      const Slot& at) const {
    const bool v = h >= p.nh + p.nkv;
    if (mine && h < p.nh) {
      store_piece(q_row + h * p.hd + lo, x);
      store_piece(q_row + h * p.hd + hi, x + VEC);
    }
    const int g = h - p.nh - (v ? p.nkv : 0);
    const bool to_cache = mine && h >= p.nh && at.values >= 0;
    const int l0 = v ? lo_v : lo, l1 = v ? hi_v : hi;
    if constexpr (QUANT) {
      if (!__any_sync(0xffffffffu, to_cache)) return;   // a warp of q heads
      float largest = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * VEC; i += 2) largest = max_abs(largest, x[i], x[i + 1]);
      uint32_t top = abs_bits(largest);
      for (int o = lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (to_cache) {
        const float scale = row_scale(top), inv = inverse(scale);
        uint8_t* o = static_cast<uint8_t*>(v ? p.kv.v : p.kv.k) + at.values + g * p.kv.head_stride;
        store_codes<VEC>(o + l0, x, inv);
        store_codes<VEC>(o + l1, x + VEC, inv);
        if (c == 0) (v ? p.sc.v : p.sc.k)[at.scale + g * p.sc.head_stride] = scale;
      }
    } else if (to_cache) {
      T* o = static_cast<T*>(v ? p.kv.v : p.kv.k) + at.values + g * p.kv.head_stride;
      store_piece(o + l0, x);
      store_piece(o + l1, x + VEC);
    }
  }
};

// Items are (token, HEADS heads); a group of lanes takes every step-th of them. The step moves it on by about 3/8 of a
// token's items each time (whole warps of them, so that a warp's stay alike): heads for the cache cost more than heads of
// q, and where the grid is a multiple of a token's items every warp would meet the same heads again and again (16 x 2048
// tokens of 32 + 8 + 8 heads: 152 us instead of 116).
// A lane without items stands at `count` and is moved on as often as the others of its warp: to less than twice the count
// and two steps, which has to stay within 32 bits.
constexpr int64_t MOST_ITEMS = (int64_t{1} << 31) - (1 << 20), MOST_STEP = 148 * WRITE_CTAS * 256;
static_assert(2 * (MOST_ITEMS + MOST_STEP) <= int64_t{1} << 32, "item numbers would wrap");
struct Items {
  unsigned count, groups, step, step_tok, step_group, item, token, group;
  __device__ __forceinline__ Items(const WriteParams& p, int lanes, unsigned n_groups) {
    const unsigned per = 256u / lanes, warp = 32u / lanes, total = gridDim.x * per;
    groups = n_groups;
    count = static_cast<unsigned>(p.tokens) * groups;
    step = total;
    if (count > total && total > groups) {
      const unsigned on = max(groups * 3 / 8 / warp * warp, warp) % groups;
      step -= (total + groups - on) % groups;
    }
    step_tok = step / groups;
    step_group = step - step_tok * groups;
    item = blockIdx.x * per + threadIdx.x / lanes;
    if (item >= step) item = count;   // the last few, for the step's sake
    token = item / groups;
    group = item - token * groups;
  }
  __device__ __forceinline__ bool left() const { return item < count; }
  __device__ __forceinline__ void advance() {
    item += step;
    token += step_tok;
    group += step_group;
    if (group >= groups) {
      group -= groups;
      ++token;
    }
  }
};

template <typename T, bool QUANT, Pairs PAIRS, int CTAS = WRITE_CTAS>
__global__ void __launch_bounds__(256, CTAS)
    rotary_write_vec_kernel(WriteParams p, int lanes, unsigned groups) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  constexpr int VEC = VALUES<T>, HEADS = WRITE_HEADS;
  __shared__ __align__(16) uint4 ahead[2][HEADS][2][256];
  const Lane<T, PAIRS> lane(p, lanes);
  const int c = lane.c, heads = lane.heads;
  Items it(p, lanes, groups);   // the item ahead
  auto fetch = [&](int to, int64_t at_pos) {
    if (it.left() && lane.owns && token_ok(p, at_pos, false)) {
      const T* row = static_cast<const T*>(p.qkv) + static_cast<int64_t>(it.token) * p.ld;
#pragma unroll
      for (int u = 0; u < HEADS; ++u) {
        const int h = it.group * HEADS + u;
        const bool v = h >= p.nh + p.nkv;
        if (h < heads) {
          copy_async16(&ahead[to][u][0][threadIdx.x], row + h * p.hd + (v ? lane.lo_v : lane.lo));
          copy_async16(&ahead[to][u][1][threadIdx.x], row + h * p.hd + (v ? lane.hi_v : lane.hi));
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // The item at hand: its token, first head, position and whether there is one; its pieces lie in ahead[buf].
  unsigned token = it.token;
  int h0 = it.group * HEADS, buf = 0;
  bool real = it.left();
  int64_t pos = real ? p.positions[token] : -1;
  fetch(0, pos);
  it.advance();
  int64_t ahead_pos = it.left() ? p.positions[it.token] : -1;
  while (__any_sync(0xffffffffu, real)) {   // all lanes of a warp stay until its last item is done
    const int64_t tok = token;
    const bool ok = real && lane.owns && token_ok(p, pos, c == 0 && h0 == 0);
    const unsigned next_token = it.token;
    const int next_h0 = it.group * HEADS;
    const int64_t next_pos = ahead_pos;
    const bool next_real = it.left();
    T* q_row = static_cast<T*>(p.q_out) + tok * p.ldq;
    Slot at = {-1, -1};
    if (ok && h0 + HEADS > p.nh) at = find_slot(p, tok, pos, c == 0 && h0 <= p.nh);
    float cs[VEC], sn[VEC];
    lane.load_turns(p, ok, pos, cs, sn);
    fetch(buf ^ 1, next_pos);
    it.advance();
    ahead_pos = it.left() ? p.positions[it.token] : -1;
    asm volatile("cp.async.wait_group 1;" ::: "memory");
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      const int h = h0 + u;
      const bool mine = ok && h < heads;
      float x[2 * VEC];
      const uint4 none = make_uint4(0, 0, 0, 0);   // lanes without pieces add zeros to the row's largest value
      unpack_piece(mine ? ahead[buf][u][0][threadIdx.x] : none, x, static_cast<const T*>(nullptr));
      unpack_piece(mine ? ahead[buf][u][1][threadIdx.x] : none, x + VEC, static_cast<const T*>(nullptr));
      if (mine && h < p.nh + p.nkv && lane.turns) lane.turn(x, cs, sn);
      lane.template put<QUANT>(p, mine, h, x, q_row, at);
    }
    token = next_token;
    h0 = next_h0;
    pos = next_pos;
    real = next_real;
    buf ^= 1;
  }
}

// STAGED: a head's values go through shared memory, where its lanes take the pairs in turn (neighbouring ones at a time,
// so that tables and banks are read in order). 8192 tokens of 32 + 8 + 8 heads of 128, 126 turned: 53 us to the 8-bit
// cache, 51 to the bf16 one, 69 in fp32, where a warp a head, as above, takes 178, 171 and 197. The whole pieces of HALVES
// take 33 to both: here an item's pieces are loaded when it begins, and nothing is on its way while they turn.
template <typename T, bool QUANT>
__global__ void __launch_bounds__(256, WRITE_CTAS)
    rotary_write_staged_kernel(WriteParams p, int lanes, unsigned groups) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  constexpr int VEC = VALUES<T>, HEADS = WRITE_HEADS;
  const Lane<T, STAGED> lane(p, lanes);
  const int c = lane.c, heads = lane.heads;
  // HEADS heads of values for the lanes of a head (`active` of them own pieces), a warp's groups of lanes apart by as many
  // banks as they have lanes.
  __shared__ __align__(16) float staged[256 * HEADS * 2 * VEC + 1024];
  const int group_floats = lanes * HEADS * 2 * VEC + (lanes < 4 ? 4 : lanes), active = p.hd / (2 * VEC);
  float* const stage = staged + threadIdx.x / lanes * group_floats;
  Items it(p, lanes, groups);
  int64_t next_pos = it.left() ? p.positions[it.token] : -1;
  while (__any_sync(0xffffffffu, it.left())) {   // all lanes of a warp stay until its last item is done
    const int h0 = it.group * HEADS;
    const int64_t tok = it.token, pos = next_pos;
    const bool ok = it.left() && lane.owns && token_ok(p, pos, c == 0 && h0 == 0);
    it.advance();
    next_pos = it.left() ? p.positions[it.token] : -1;
    const T* row = static_cast<const T*>(p.qkv) + tok * p.ld;
    T* q_row = static_cast<T*>(p.q_out) + tok * p.ldq;
    Slot at = {-1, -1};
    if (ok && h0 + HEADS > p.nh) at = find_slot(p, tok, pos, c == 0 && h0 <= p.nh);
    float cs[VEC], sn[VEC];
    lane.load_turns(p, ok, pos, cs, sn);
    uint4 raw[HEADS][2];
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      raw[u][0] = raw[u][1] = make_uint4(0, 0, 0, 0);
      if (ok && h0 + u < heads) {
        raw[u][0] = *reinterpret_cast<const uint4*>(row + (h0 + u) * p.hd + lane.lo);
        raw[u][1] = *reinterpret_cast<const uint4*>(row + (h0 + u) * p.hd + lane.hi);
      }
    }
    // A lane's own pieces go in and come out; between the barriers the pairs turn where they lie.
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      float x[2 * VEC];
      unpack_piece(raw[u][0], x, static_cast<const T*>(nullptr));
      unpack_piece(raw[u][1], x + VEC, static_cast<const T*>(nullptr));
      if (ok) {
        put_floats<VEC>(stage + u * lanes * 2 * VEC + lane.lo, x);
        put_floats<VEC>(stage + u * lanes * 2 * VEC + lane.hi, x + VEC);
      }
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      float* s = stage + u * lanes * 2 * VEC + c;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (ok && h0 + u < p.nh + p.nkv && c + active * i < lane.half) {
          const float a0 = s[active * i], b0 = s[active * i + lane.half];
          s[active * i] = a0 * cs[i] - b0 * sn[i];
          s[active * i + lane.half] = b0 * cs[i] + a0 * sn[i];
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < HEADS; ++u) {
      float x[2 * VEC] = {};   // lanes without pieces add zeros to the row's largest value
      if (ok) {
        load_floats<VEC>(stage + u * lanes * 2 * VEC + lane.lo, x);
        load_floats<VEC>(stage + u * lanes * 2 * VEC + lane.hi, x + VEC);
      }
      lane.template put<QUANT>(p, ok && h0 + u < heads, h0 + u, x, q_row, at);
    }
  }
}

// Whole 16-byte pieces everywhere: heads of 2 VEC values' multiples, rows, tables and cache on their boundaries.
template <typename T>
bool write_vec_ok(const WriteParams& p, bool quant) {
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  if (p.hd % (2 * VEC) || p.hd > 64 * VEC ) return false;
  const int64_t el = quant ? 16 : VEC;   // elements of the cache in 16 bytes
  if (p.ld % VEC || (p.nh > 0 && p.ldq % VEC) || p.kv.block_stride % el || p.kv.head_stride % el) return false;
  if (quant && p.hd % 16) return false;
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.qkv) | (p.nh > 0 ? reinterpret_cast<uintptr_t>(p.q_out) : 0) |
                        (p.rd > 0 ? reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t) : 0) |
                        reinterpret_cast<uintptr_t>(p.kv.k) | reinterpret_cast<uintptr_t>(p.kv.v);
  return (all & 15) == 0;
}

// Flags the bad blocks of a read-back for given queries: those that one of their row's T positions reaches. Table columns
// that no query looks at may hold anything. One thread a column; only a bad block's looks through the positions. A kernel of
// its own: the same test inside the read-back cost that one 4 to 9 % by its registers.
__global__ void __launch_bounds__(256)
    flag_seen_blocks_kernel(KVCache kv, int64_t cols, const int64_t* __restrict__ positions, int T, unsigned* err) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads other kernels' data
  const int64_t col = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x, r = blockIdx.y;
  if (col >= cols) return;
  const int64_t blk = kv.table[r * kv.table_stride + col];
  if (blk >= 0 && blk < kv.num_blocks) return;
  bool seen = false;
  for (int t = 0; t < T && !seen; ++t) seen = positions[r * T + t] >= col * kv.block_size;
  if (seen) flag_error(err, ERR_BAD_SLOT);
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

// The vector form: heads of whole VEC-value pieces, 16 bytes of each output at a time. One wave of CTAs stays and takes
// chunks of 256 / (hd / VEC) slots of a (row, head) in turn; many small CTAs an SM (8) beat more loads a thread (8 rows of
// 16384 slots of 8 x 128: 139 us, 89 % of HBM; two slots a thread 141 at 6 CTAs, a CTA for every chunk 165).
constexpr int DEQUANT_CTAS = 8;
template <typename T>
__global__ void __launch_bounds__(256, DEQUANT_CTAS)
    kv_dequant_vec_kernel(KVCache kv, KVScales sc, uint32_t n_slots, int nkv, int hd, T* __restrict__ k_out,
                          T* __restrict__ v_out, unsigned* err, unsigned chunks, unsigned total) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  constexpr int VEC = 16 / static_cast<int>(sizeof(T));
  const int lanes = hd / VEC, rows = 256 / lanes, c = threadIdx.x % lanes, i = threadIdx.x / lanes;
  if (i >= rows) return;
  for (unsigned item = blockIdx.x; item < total; item += gridDim.x) {
    const unsigned rg = item / chunks, r = rg / nkv, g = rg - r * nkv;
    const uint32_t s = (item - rg * chunks) * rows + i;
    if (s >= n_slots) continue;
    int64_t col, in;
    split_slot(s, kv.block_size, col, in);
    const int64_t blk = col < kv.table_cols ? kv.table[r * kv.table_stride + col] : -1;
    uint2 ck = make_uint2(0, 0), cv = ck;
    float sk = 0.f, sv = 0.f;
    if (blk >= 0 && blk < kv.num_blocks) {
      const int64_t at = blk * kv.block_stride + g * kv.head_stride + in * hd + c * VEC;
      const int64_t sat = blk * sc.block_stride + g * sc.head_stride + in;
      ck = load_codes<VEC>(static_cast<const uint8_t*>(kv.k) + at);
      cv = load_codes<VEC>(static_cast<const uint8_t*>(kv.v) + at);
      sk = sc.k[sat];
      sv = sc.v[sat];
    } else if (c == 0 && in == 0) {
      flag_error(err, ERR_BAD_SLOT);
    }
    const int64_t o = (static_cast<int64_t>(rg) * n_slots + s) * hd + c * VEC;
    float x[VEC];
    decode_piece<VEC>(ck, sk, x);
    store_piece(k_out + o, x);
    decode_piece<VEC>(cv, sv, x);
    store_piece(v_out + o, x);
  }
}

template <typename T>
int write_t(const WriteParams& p, bool quant, int interleaved, cudaStream_t st) {
  constexpr int PIECES = 32 / static_cast<int>(sizeof(T));   // values a lane of the vector form holds of a head
  int lanes = 1;
  while (lanes * PIECES < p.hd) lanes *= 2;
  const int64_t vec_items = p.tokens * ((p.nh + 2 * p.nkv + 1) / 2) * lanes;   // thread numbers
  if (write_vec_ok<T>(p, quant) && vec_items <= MOST_ITEMS) {
    const unsigned groups = (p.nh + 2 * p.nkv + WRITE_HEADS - 1) / WRITE_HEADS;
    const int64_t blocks = (p.tokens * groups * lanes + 255) / 256;
    auto launch = [&](auto kernel, int ctas) {
      const int64_t wave = 148 * ctas;
      launch_pdl_async(kernel, static_cast<unsigned>(blocks < wave ? blocks : wave), 256, 0, st, p, lanes, groups);
    };
    // A plain write past L2 (a lane reads 64 bytes an item) takes two CTAs an SM, with registers for more loads at once and
    // fewer streams on HBM: 16384 tokens of 32 + 8 + 8 heads 65 us against 70 with three, 65536 249 against 281; 8192 34.5
    // against 33.5. The 8-bit cache's needs the third for its arithmetic (16 x 2048 tokens: 116 us, 130 with two).
    const bool large = p.tokens * groups * lanes > (int64_t{128} << 20) / 64;
    if (!interleaved && p.rd % PIECES)
      launch(quant ? rotary_write_staged_kernel<T, true> : rotary_write_staged_kernel<T, false>, WRITE_CTAS);
    else if (quant)
      launch(interleaved ? rotary_write_vec_kernel<T, true, NEIGHBOURS> : rotary_write_vec_kernel<T, true, HALVES>,
             WRITE_CTAS);
    else if (!large)
      launch(interleaved ? rotary_write_vec_kernel<T, false, NEIGHBOURS> : rotary_write_vec_kernel<T, false, HALVES>,
             WRITE_CTAS);
    else
      launch(interleaved ? rotary_write_vec_kernel<T, false, NEIGHBOURS, 2> : rotary_write_vec_kernel<T, false, HALVES, 2>,
             2);
    return check_launch("rotary_write_vec_kernel");
  }
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
               const int64_t* positions, int64_t T_new, void* k_out, void* v_out, cudaStream_t st) {
  unsigned* err = error_word();
  if (!err) return -1;
  if (positions) {
    const int64_t cols = (n_slots - 1) / kv.block_size + 1;
    const dim3 grid(static_cast<unsigned>((cols + 255) / 256), static_cast<unsigned>(B));
    launch_pdl_async(flag_seen_blocks_kernel, grid, 256, 0, st, kv, cols, positions, static_cast<int>(T_new), err);
    if (check_launch("flag_seen_blocks_kernel")) return -1;
    err = nullptr;   // the read-back itself reports nothing
  }
  const int vec = dtype == F32 ? 4 : 8;
  const uintptr_t out = reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out);
  const uintptr_t in = reinterpret_cast<uintptr_t>(kv.k) | reinterpret_cast<uintptr_t>(kv.v);
  const bool pieces = hd % vec == 0 && hd <= 256 * vec && (out & 15) == 0 && (in & (vec - 1)) == 0 &&
                      kv.block_stride % vec == 0 && kv.head_stride % vec == 0;
  if (pieces) {
    const int64_t rows = 256 / (hd / vec), chunks = (n_slots + rows - 1) / rows, total = chunks * B * nkv;
    if (total > INT32_MAX) return fail("fs_kv_dequant: too many slots");
    const unsigned ctas = static_cast<unsigned>(total < 148 * DEQUANT_CTAS ? total : 148 * DEQUANT_CTAS);
    if (dtype == F32)
      launch_pdl_async(kv_dequant_vec_kernel<float>, ctas, 256, 0, st, kv, sc, static_cast<uint32_t>(n_slots),
                       static_cast<int>(nkv), static_cast<int>(hd), static_cast<float*>(k_out),
                       static_cast<float*>(v_out), err, static_cast<unsigned>(chunks), static_cast<unsigned>(total));
    else
      launch_pdl_async(kv_dequant_vec_kernel<__nv_bfloat16>, ctas, 256, 0, st, kv, sc, static_cast<uint32_t>(n_slots),
                       static_cast<int>(nkv), static_cast<int>(hd), static_cast<__nv_bfloat16*>(k_out),
                       static_cast<__nv_bfloat16*>(v_out), err, static_cast<unsigned>(chunks), static_cast<unsigned>(total));
    return check_launch("kv_dequant_vec_kernel");
  }
  const dim3 grid(static_cast<unsigned>((n_slots * hd + 255) / 256), static_cast<unsigned>(nkv),
                  static_cast<unsigned>(B));
  auto run = [&](auto* k, auto* v) {
    using T = std::remove_pointer_t<decltype(k)>;
    launch_pdl_async(kv_dequant_kernel<T>, grid, 256, 0, st, kv, sc, static_cast<uint32_t>(n_slots),
                     static_cast<int>(nkv), static_cast<int>(hd), k, v, err);
  };
  if (dtype == F32)
    run(static_cast<float*>(k_out), static_cast<float*>(v_out));
  else
    run(static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out));
  return check_launch("kv_dequant_kernel");
}

}  // namespace fs
