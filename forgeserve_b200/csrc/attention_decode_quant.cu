// Decode attention (one new query per row) over the 8-bit cache of kv_quant.cu: grouped query heads, slot s of a row
// visible iff s <= position and s < n_slots, scale 1/sqrt(hd), as attention_decode.cu over an unquantised cache.
//
// With codes kq, vq and scales ks, vs of a (slot, KV head) row:
//     s_j = (q . kq_j) ks_j scale,   p_j = exp(s_j - max s),   out = sum_j p_j vs_j vq_j / sum_j p_j
// so a scale is one factor on a score or on a probability, and the products run on the codes themselves.
// The floor is the cache's bytes: 2 (hd + 4) for each visible slot of each KV head, read once for all its query heads.
//
// A row's slots are cut into splits of SPLIT_KEYS, one CTA each, whatever the batch and the table's width, so the order
// of the sums depends on the row alone (a step gives the same bits eagerly, in a CUDA graph with a padded table, or in
// micro-batches); quant_combine_kernel joins the splits. Workspace (fp32): sums [B][nh][splits][hd], then (max, sum)
// [B][nh][splits][2] in the log2 domain.
//
// A row with a negative position sees nothing and gets zeros. A block number outside the cache reads as zero rows and
// flags ERR_BAD_SLOT. Scores of -infinity weigh nothing; a row whose scores all are, or that meets a NaN or +infinity,
// gives NaN, as the formula does.
#include <string>

#include "common.cuh"
#include "kernels.h"
#include "quant.cuh"

namespace fs {
namespace decode_quant {

namespace {

constexpr int SPLIT_KEYS = 512;
constexpr int HEADS = 8;   // query heads of one KV head that a CTA handles

struct Params {
  const void* q;
  int64_t ldq;
  KVCache kv;
  KVScales sc;
  int64_t n_slots;
  const int64_t* positions;
  void* out;
  int64_t ldo;
  int nh, rep, hd, splits, groups;   // groups: CTAs a KV head, of HEADS query heads each
  float scale_log2;
  float* ws;
  unsigned* err;
};

__device__ __forceinline__ int64_t visible(const Params& p, int64_t r) {
  const int64_t pos = p.positions[r];
  return pos < 0 ? 0 : (pos < p.n_slots ? pos + 1 : p.n_slots);
}

// max that an exponent may be taken against: -infinity (no finite score) becomes 0, so that exp2(-inf - m) is 0.
__device__ __forceinline__ float safe_max(float m) { return m == -INFINITY ? 0.f : m; }

// Any type, hd (<= 256) and layout: 32 keys at a time as fp32 in shared memory; a warp owns two query heads, a lane
// one key of the scores and hd / 32 dims of the sums.
template <typename T>
__global__ void __launch_bounds__(128) quant_decode_kernel(Params p) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  constexpr int CHUNK = 32, MAXD = 8;
  extern __shared__ float sm[];
  const int hd = p.hd, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* ks = sm;                          // [CHUNK][hd + 1]
  float* vs = ks + CHUNK * (hd + 1);       // [CHUNK][hd]
  float* qs = vs + CHUNK * hd;             // [HEADS][hd]
  __shared__ int64_t at[CHUNK];
  __shared__ float ksc[CHUNK], vsc[CHUNK];

  const int split = blockIdx.x, g = blockIdx.y / p.groups, h0 = (blockIdx.y % p.groups) * HEADS;
  const int64_t r = blockIdx.z;
  const int heads = p.rep - h0 < HEADS ? p.rep - h0 : HEADS;
  const int64_t n_vis = visible(p, r);
  const int64_t begin = static_cast<int64_t>(split) * SPLIT_KEYS;
  const int64_t end = begin + SPLIT_KEYS < n_vis ? begin + SPLIT_KEYS : n_vis;
  if (begin >= n_vis && !(p.splits == 1 && n_vis == 0)) return;   // the join does not read an empty split

  for (int i = tid; i < heads * hd; i += blockDim.x)
    qs[i] = to_f(static_cast<const T*>(p.q)[r * p.ldq + static_cast<int64_t>(g * p.rep + h0) * hd + i]);
  float acc[2][MAXD], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < MAXD; ++i) acc[t][i] = 0.f;

  for (int64_t c0 = begin; c0 < end; c0 += CHUNK) {
    const int n = static_cast<int>(end - c0 < CHUNK ? end - c0 : CHUNK);
    __syncthreads();
    if (tid < n) {
      int64_t col, in;
      split_slot(c0 + tid, p.kv.block_size, col, in);
      const int64_t blk = col < p.kv.table_cols ? p.kv.table[r * p.kv.table_stride + col] : -1;
      const bool ok = blk >= 0 && blk < p.kv.num_blocks;
      if (!ok) flag_error(p.err, ERR_BAD_SLOT);
      const int64_t sat = blk * p.sc.block_stride + g * p.sc.head_stride + in;
      at[tid] = ok ? blk * p.kv.block_stride + g * p.kv.head_stride + in * hd : -1;
      ksc[tid] = ok ? p.sc.k[sat] : 0.f;
      vsc[tid] = ok ? p.sc.v[sat] : 0.f;
    }
    __syncthreads();
    for (int i = tid; i < n * hd; i += blockDim.x) {
      const int key = i / hd, d = i - key * hd;
      const int64_t o = at[key];
      ks[key * (hd + 1) + d] = o < 0 ? 0.f : e4m3_to_f(static_cast<const uint8_t*>(p.kv.k)[o + d]);
      vs[i] = o < 0 ? 0.f : e4m3_to_f(static_cast<const uint8_t*>(p.kv.v)[o + d]) * vsc[key];
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int h = warp + 4 * t;
      if (h >= heads) break;
      float s = -INFINITY;
      if (lane < n) {
        s = 0.f;
        for (int d = 0; d < hd; ++d) s = fmaf(qs[h * hd + d], ks[lane * (hd + 1) + d], s);
        s *= ksc[lane] * p.scale_log2;
      }
      float top = s;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float mn = fmaxf(m[t], top);
      const float corr = exp2f(m[t] - safe_max(mn)), pr = lane < n ? exp2f(s - safe_max(mn)) : 0.f;
      m[t] = mn;
      l[t] = l[t] * corr + pr;
#pragma unroll
      for (int i = 0; i < MAXD; ++i) acc[t][i] *= corr;
      for (int k = 0; k < n; ++k) {
        const float pk = __shfl_sync(0xffffffffu, pr, k);
#pragma unroll
        for (int i = 0; i < MAXD; ++i)
          if (lane + 32 * i < hd) acc[t][i] = fmaf(pk, vs[k * hd + lane + 32 * i], acc[t][i]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int h = warp + 4 * t;
    if (h >= heads) break;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l[t] += __shfl_xor_sync(0xffffffffu, l[t], o);
    const int hh = g * p.rep + h0 + h;
    const int64_t part = (r * p.nh + hh) * p.splits + split;
#pragma unroll
    for (int i = 0; i < MAXD; ++i) {
      const int d = lane + 32 * i;
      if (d >= hd) break;
      if (p.splits == 1)
        static_cast<T*>(p.out)[r * p.ldo + static_cast<int64_t>(hh) * hd + d] =
            from_f<T>(n_vis == 0 ? 0.f : acc[t][i] / l[t]);
      else
        p.ws[part * hd + d] = acc[t][i];
    }
    if (p.splits > 1 && lane == 0) {
      float* ml = p.ws + static_cast<int64_t>(gridDim.z) * p.nh * p.splits * hd + 2 * part;
      ml[0] = m[t];
      ml[1] = l[t];
    }
  }
}

// ------------------------------------------------------------------------------------ tensor-core kernel
// hd 64, 128 or 256, 16-byte rows. The codes are exact in f16, so both products run as mma.sync m16n8k16 f16 with fp32
// sums and the scales never touch them:
//     S^T (16 keys x 8 heads) = K (16 x hd) Q^T (hd x 8),   O^T (hd x 8 heads) += V^T (hd x 16) P^T (16 x 8)
// with the query heads of the KV head as the N side (NT tiles of 8). A contraction's index order is free as long as
// both operands agree, and so are the rows of O^T; they are chosen so that every lane's operand values are 16
// neighbouring bytes of a cache row: lane (g, t) = (lane / 4, lane % 4) takes, of keys g and g + 8, the 16-byte chunks
// t, t + 4, .. for K, and of keys 2t, 2t+1, 2t+8, 2t+9 the bytes g hd/8 .. + hd/8 for V. So a lane copies exactly the
// bytes it will use (cp.async, whole sectors) into slots of its own: a ring in shared memory without barriers, ldmatrix
// or swizzles, and any block size. P^T reaches the B layout by movmatrix.
//
// Q enters as f16 after a scale by a power of two that brings each head's largest |q| to [1, 2): exact for bf16 down to
// 2^-14 of it, off by 2^-25 of it below. fp32 queries enter as two halves (a value and its remainder times 2^11): 22
// bits. P enters as p_j vs_j against a running maximum of its own, so that values whose scales differ widely keep the
// f16 range: vs = mantissa 2^e, P = exp2(s + e - mo) mantissa, mo >= max(s + e) - SLACK. bf16 rounds P to f16 (2^-11); fp32
// adds its remainder as a second product. Maxima are raised only when a score exceeds them by SLACK = 2^8: one vote
// a tile instead of a reduction.
namespace tc {

constexpr int WARPS = 4, TILE = 16, TILES = SPLIT_KEYS / TILE / WARPS;   // tiles a warp has of a full split
constexpr float SLACK = 8.f;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// BYTES (4, 8 or 16) from global to shared memory, zeros where !ok.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? BYTES : 0;
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ uint32_t lo_pair(uint32_t w) { return e4m3x2_to_half2(static_cast<uint16_t>(w)); }
__device__ __forceinline__ uint32_t hi_pair(uint32_t w) { return e4m3x2_to_half2(static_cast<uint16_t>(w >> 16)); }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^x, 2^-22 of the value off at most; results below 2^-126 are zero.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// vs as mantissa * 2^e; zero gives e = -infinity, infinity and NaN themselves. Scales are not negative.
__device__ __forceinline__ void split_scale(float vs, float& e, float& mant) {
  const uint32_t b = __float_as_uint(vs);
  if (b - 0x00800000u < 0x7f000000u) {
    e = static_cast<float>(static_cast<int>(b >> 23) - 127);
    mant = __uint_as_float((b & 0x007fffffu) | 0x3f800000u);
  } else {
    e = log2f(vs);
    mant = 1.f;
  }
}

// WHOLE: the block size is a multiple of 16, so a tile lies in one block and its rows follow one another; otherwise
// every key is looked up by itself.
template <typename T, int HD, int NT, bool WHOLE>
struct Geo {
  static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;        // f16 terms of q and of p
  static constexpr int KS = HD / 16;                          // k steps of S^T, and m tiles of O^T
  static constexpr int KC = HD / 64;                          // 16-byte chunks a lane takes of a K row
  static constexpr int VB = HD / 8 < 16 ? 8 : 16;             // bytes of one V copy
  static constexpr int VC = HD / 8 / VB;                      // V copies a key
  static constexpr int STAGES = 2;
  static constexpr bool Q_REGS = NT * PARTS * KS <= 8;        // q's operands in registers, else read from shared memory
  static constexpr int V_OFF = 2 * KC * 512;                  // slot: K copies, V copies (32 lanes each), 32 scales
  static constexpr int S_OFF = V_OFF + 4 * VC * VB * 32;
  static constexpr int SLOT = S_OFF + 128;
  static constexpr int RING = WARPS * STAGES * SLOT;
  static constexpr int Q_OFF = RING;                          // q as B operands: [NT][PARTS][KS][32 lanes] of 8 bytes
  static constexpr int Q_BYTES = NT * PARTS * KS * 256;
  static constexpr int AT_OFF = Q_OFF + Q_BYTES;              // offsets of a warp's tiles or keys: values, then scales
  static constexpr int AT_N = WARPS * TILES * (WHOLE ? 1 : TILE);
  static constexpr int H_OFF = AT_OFF + AT_N * 16;            // [8 NT] score factors
  static constexpr int O_ROW = HD + 4;                        // padded: the lanes' writes spread over the banks
  static constexpr int O_BYTES = WARPS * 8 * NT * (O_ROW + 2) * 4;   // the warps' sums, then (max, sum), over all that
  static constexpr int SMEM = O_BYTES > H_OFF + 32 * NT ? O_BYTES : H_OFF + 32 * NT;
};

template <typename T, int HD, int NT, bool WHOLE>
__global__ void __launch_bounds__(32 * WARPS) quant_decode_tc_kernel(Params p) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  using G = Geo<T, HD, NT, WHOLE>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, tl = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y / p.groups, h0 = (blockIdx.y % p.groups) * 8 * NT;
  const int64_t r = blockIdx.z;
  const int heads = p.rep - h0 < 8 * NT ? p.rep - h0 : 8 * NT;
  const int64_t n_vis = visible(p, r);
  const int64_t begin = static_cast<int64_t>(split) * SPLIT_KEYS;
  if (begin >= n_vis) {
    if (p.splits == 1)   // a row that sees nothing
      for (int i = threadIdx.x; i < heads * HD; i += blockDim.x)
        static_cast<T*>(p.out)[r * p.ldo + static_cast<int64_t>(kvh * p.rep + h0) * HD + i] = from_f<T>(0.f);
    return;              // the join does not read an empty split
  }
  const int n_keys = static_cast<int>(n_vis - begin < SPLIT_KEYS ? n_vis - begin : SPLIT_KEYS);
  const int n_tiles = (n_keys + TILE - 1) / TILE;
  const int my_n = n_tiles > warp ? (n_tiles - warp + WARPS - 1) / WARPS : 0;   // tiles warp, warp + 4, ..

  // Where this warp's tiles (or keys) begin, -1 for a key that is not visible or whose block is bad.
  constexpr int PER = WHOLE ? 1 : TILE, LOOK = TILES * PER;
  int64_t* at = reinterpret_cast<int64_t*>(smem + G::AT_OFF) + warp * LOOK;
  int64_t* sat = at + WARPS * LOOK;
#pragma unroll
  for (int i = 0; i < (LOOK + 31) / 32; ++i) {
    const int k = lane + 32 * i, key = (warp + WARPS * (k / PER)) * TILE + k % PER;
    int64_t a = -1, b = -1;
    if (key < n_keys && k < LOOK) {
      int64_t col, in;
      split_slot(begin + key, p.kv.block_size, col, in);
      const int64_t blk = col < p.kv.table_cols ? p.kv.table[r * p.kv.table_stride + col] : -1;
      if (blk >= 0 && blk < p.kv.num_blocks) {
        a = blk * p.kv.block_stride + kvh * p.kv.head_stride + in * HD;
        b = blk * p.sc.block_stride + kvh * p.sc.head_stride + in;
      } else {
        flag_error(p.err, ERR_BAD_SLOT);
      }
    }
    if (k < LOOK) {
      at[k] = a;
      sat[k] = b;
    }
  }
  __syncwarp();

  const uint8_t* kbase = static_cast<const uint8_t*>(p.kv.k);
  const uint8_t* vbase = static_cast<const uint8_t*>(p.kv.v);
  const float* sbase = lane < TILE ? p.sc.k : p.sc.v;
  uint8_t* ring = smem + warp * G::STAGES * G::SLOT;
  auto issue = [&](int j) {   // tile j of this warp into slot j % STAGES
    const uint32_t slot = smem_u32(ring) + (j % G::STAGES) * G::SLOT;
    const uint32_t dst = slot + lane * 16, vdst = slot + G::V_OFF + lane * G::VB;
    if constexpr (WHOLE) {
      const int64_t o = at[j], so = sat[j];
      const int n = o < 0 ? 0 : n_keys - (warp + WARPS * j) * TILE;   // rows to read; the rest become zeros
      const uint8_t* kp = kbase + (o < 0 ? 0 : o) + tl * 16;
      const uint8_t* vp = vbase + (o < 0 ? 0 : o) + gl * (HD / 8);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool ok = gl + 8 * i < n;
        const uint8_t* src = ok ? kp + (gl + 8 * i) * HD : kbase;
#pragma unroll
        for (int c = 0; c < G::KC; ++c) copy_async<16>(dst + (i * G::KC + c) * 512, src + c * 64, ok);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * tl + (i & 1) + 8 * (i >> 1);
        const bool ok = key < n;
        const uint8_t* src = ok ? vp + key * HD : vbase;
#pragma unroll
        for (int c = 0; c < G::VC; ++c)
          copy_async<G::VB>(vdst + (i * G::VC + c) * 32 * G::VB, src + c * G::VB, ok);
      }
      const bool ok = (lane & (TILE - 1)) < n;
      copy_async<4>(slot + G::S_OFF + lane * 4, sbase + (ok ? so + (lane & (TILE - 1)) : 0), ok);
    } else {
      const int64_t* a = at + j * TILE;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t o = a[gl + 8 * i];
#pragma unroll
        for (int c = 0; c < G::KC; ++c)
          copy_async<16>(dst + (i * G::KC + c) * 512, kbase + (o < 0 ? 0 : o + (tl + 4 * c) * 16), o >= 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t o = a[2 * tl + (i & 1) + 8 * (i >> 1)];
#pragma unroll
        for (int c = 0; c < G::VC; ++c)
          copy_async<G::VB>(vdst + (i * G::VC + c) * 32 * G::VB, vbase + (o < 0 ? 0 : o + gl * (HD / 8) + c * G::VB),
                            o >= 0);
      }
      const int64_t so = sat[j * TILE + (lane & (TILE - 1))];
      copy_async<4>(slot + G::S_OFF + lane * 4, sbase + (so < 0 ? 0 : so), so >= 0);
    }
  };
#pragma unroll
  for (int j = 0; j < G::STAGES; ++j) {
    if (j < my_n) issue(j);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // Q: warp w scales heads w, w + 4, .. to [1, 2) and lays them out as the lanes' B operands.
  float* hs = reinterpret_cast<float*>(smem + G::H_OFF);
  for (int h = warp; h < 8 * NT; h += WARPS) {
    float x[HD / 32];
    uint32_t top = 0;
    const bool real = h < heads;
    const T* q = static_cast<const T*>(p.q) + r * p.ldq + static_cast<int64_t>(kvh * p.rep + h0 + h) * HD;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      x[i] = real ? to_f(q[lane + 32 * i]) : 0.f;
      top = max(top, abs_bits(x[i]));
    }
    // 2^-e of the largest value as two factors, each inside fp32's range
    top = __reduce_max_sync(0xffffffffu, top);
    const int e = top < 0x00800000u ? (top ? -126 : 0) : static_cast<int>(top >> 23) - 127;
    const int e0 = e >> 1, e1 = e - e0;
    const float f0 = __int_as_float((127 - e0) << 23), f1 = __int_as_float((127 - e1) << 23);
    __half* dst = reinterpret_cast<__half*>(smem + G::Q_OFF) + static_cast<int64_t>(h >> 3) * G::PARTS * G::KS * 128;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int d = lane + 32 * i, c = d >> 4;
      const int idx = (((c >> 2) * 4 + ((d & 15) >> 2)) * 32 + (h & 7) * 4 + (c & 3)) * 4 + (d & 3);
      const float y = x[i] * f0 * f1;
      const __half hi = __float2half_rn(y);
      dst[idx] = hi;
      if constexpr (G::PARTS == 2) dst[G::KS * 128 + idx] = __float2half_rn((y - __half2float(hi)) * 2048.f);
    }
    if (lane == 0) hs[h] = p.scale_log2 * __int_as_float((127 + e0) << 23) * __int_as_float((127 + e1) << 23);
  }
  __syncthreads();
  const uint2* qf = reinterpret_cast<const uint2*>(smem + G::Q_OFF) + lane;
  uint2 qr[G::Q_REGS ? NT * G::PARTS * G::KS : 1];
  if constexpr (G::Q_REGS)
#pragma unroll
    for (int i = 0; i < NT * G::PARTS * G::KS; ++i) qr[i] = qf[i * 32];

  // This lane's columns are heads 8 n + 2 tl and + 1 of each N tile n.
  // ms and mos are the maxima as exponents are taken against them (safe_max).
  float fs[NT][2], m[NT][2], mo[NT][2], ms[NT][2], mos[NT][2], l[NT][2], acc[NT][G::KS][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      fs[n][c] = hs[8 * n + 2 * tl + c];
      m[n][c] = mo[n][c] = -INFINITY;
      ms[n][c] = mos[n][c] = l[n][c] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < G::KS; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
  }

  for (int j = 0; j < my_n; ++j) {
    asm volatile("cp.async.wait_group %0;" ::"n"(G::STAGES - 1) : "memory");
    __syncwarp();   // the other lanes' scales
    const uint8_t* slot = ring + (j % G::STAGES) * G::SLOT;
    const float* sc = reinterpret_cast<const float*>(slot + G::S_OFF);
    const int k0 = (warp + WARPS * j) * TILE;
    float s[NT][4];
    {
      // two chains of products, so that one's latency covers the other's
      float a[NT][G::PARTS][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < G::PARTS; ++q)
#pragma unroll
          for (int c = 0; c < 8; ++c) a[n][q][c >> 2][c & 3] = 0.f;
#pragma unroll
      for (int c = 0; c < G::KC; ++c) {
        const uint4 u = *reinterpret_cast<const uint4*>(slot + c * 512 + lane * 16);
        const uint4 w = *reinterpret_cast<const uint4*>(slot + (G::KC + c) * 512 + lane * 16);
        const uint32_t ku[4] = {u.x, u.y, u.z, u.w}, kw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = lo_pair(ku[i]), a1 = lo_pair(kw[i]), a2 = hi_pair(ku[i]), a3 = hi_pair(kw[i]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < G::PARTS; ++q) {
              const int at_q = (n * G::PARTS + q) * G::KS + c * 4 + i;
              const uint2 b = G::Q_REGS ? qr[G::Q_REGS ? at_q : 0] : qf[at_q * 32];
              mma_f16(a[n][q][i & 1], a0, a1, a2, a3, b.x, b.y);
            }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[n][c] = a[n][0][0][c] + a[n][0][1][c];
          if constexpr (G::PARTS == 2) s[n][c] = fmaf(a[n][1][0][c] + a[n][1][1][c], 1.f / 2048.f, s[n][c]);
        }
    }
    // Scores of keys gl (c 0, 1) and gl + 8 (c 2, 3), log2 domain; u: with the exponent of the value's scale.
    const bool in0 = k0 + gl < n_keys, in1 = k0 + gl + 8 < n_keys;
    float e[2], mant[2];
    split_scale(sc[TILE + gl], e[0], mant[0]);
    split_scale(sc[TILE + gl + 8], e[1], mant[1]);
    const float ks[2] = {sc[gl], sc[gl + 8]};
    bool raise = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        s[n][c] = (c < 2 ? in0 : in1) ? s[n][c] * (fs[n][c & 1] * ks[c >> 1]) : -INFINITY;
        raise |= s[n][c] > m[n][c & 1] + SLACK || s[n][c] + e[c >> 1] > mo[n][c & 1] + SLACK;
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float t = fmaxf(s[n][c], s[n][c + 2]), u = fmaxf(s[n][c] + e[0], s[n][c + 2] + e[1]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
            u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, o));
          }
          t = fmaxf(t, m[n][c]);
          u = fmaxf(u, mo[n][c]);
          ms[n][c] = safe_max(t);
          mos[n][c] = safe_max(u);
          const float cl = ex2(m[n][c] - ms[n][c]), co = ex2(mo[n][c] - mos[n][c]);
          l[n][c] *= cl;
#pragma unroll
          for (int i = 0; i < G::KS; ++i) {
            acc[n][i][c] *= co;
            acc[n][i][c + 2] *= co;
          }
          m[n][c] = t;
          mo[n][c] = u;
        }
    }
    uint32_t pb[NT][G::PARTS][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool in = c < 2 ? in0 : in1;
        l[n][c & 1] += in ? ex2(s[n][c] - ms[n][c & 1]) : 0.f;
        w[c] = in ? ex2(s[n][c] + e[c >> 1] - mos[n][c & 1]) * mant[c >> 1] : 0.f;
      }
      const uint32_t p0 = pack_half2(w[0], w[1]), p1 = pack_half2(w[2], w[3]);
      pb[n][0][0] = movmatrix_trans(p0);
      pb[n][0][1] = movmatrix_trans(p1);
      if constexpr (G::PARTS == 2) {
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&p0));
        const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
        pb[n][1][0] = movmatrix_trans(pack_half2(w[0] - f0.x, w[1] - f0.y));
        pb[n][1][1] = movmatrix_trans(pack_half2(w[2] - f1.x, w[3] - f1.y));
      }
    }
    // V: words of four dims of this lane's four keys, paired by key.
    const uint8_t* vs = slot + G::V_OFF + lane * G::VB;
#pragma unroll
    for (int c = 0; c < G::VC; ++c) {
      uint32_t v[4][G::VB / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* src = vs + (i * G::VC + c) * 32 * G::VB;
        if constexpr (G::VB == 16) {
          const uint4 u = *reinterpret_cast<const uint4*>(src);
          v[i][0] = u.x, v[i][1] = u.y, v[i][2] = u.z, v[i][3] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
          v[i][0] = u.x, v[i][1] = u.y;
        }
      }
#pragma unroll
      for (int w = 0; w < G::VB / 4; ++w)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t sel = half ? 0x7362u : 0x5140u;
          const uint32_t x = __byte_perm(v[0][w], v[1][w], sel), y = __byte_perm(v[2][w], v[3][w], sel);
          const uint32_t a0 = lo_pair(x), a1 = hi_pair(x), a2 = lo_pair(y), a3 = hi_pair(y);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < G::PARTS; ++q)
              mma_f16(acc[n][(c * (G::VB / 4) + w) * 2 + half], a0, a1, a2, a3, pb[n][q][0], pb[n][q][1]);
        }
    }
    __syncwarp();   // every lane has read the slot's scales
    if (j + G::STAGES < my_n) issue(j + G::STAGES);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // Merge the warps: sums against max m, through shared memory.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
  __syncthreads();   // ring, q and offsets are free
  float* osm = reinterpret_cast<float*>(smem);                     // [WARPS][8 NT][O_ROW]
  float* msm = osm + WARPS * 8 * NT * G::O_ROW;                    // [WARPS][8 NT][2]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int h = warp * 8 * NT + 8 * n + 2 * tl + c;
      const float f = exp2f(mos[n][c] - ms[n][c]);
#pragma unroll
      for (int i = 0; i < G::KS; ++i)
        *reinterpret_cast<float2*>(osm + h * G::O_ROW + gl * (HD / 8) + 2 * i) =
            make_float2(acc[n][i][c] * f, acc[n][i][c + 2] * f);
      if (gl == 0) {
        msm[2 * h] = m[n][c];
        msm[2 * h + 1] = l[n][c];
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * HD; i += blockDim.x) {
    const int h = i / HD, d = i % HD;
    float top = -INFINITY, total = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, msm[2 * (w * 8 * NT + h)]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2f(msm[2 * (w * 8 * NT + h)] - safe_max(top));
      total += f * msm[2 * (w * 8 * NT + h) + 1];
      o += f * osm[(w * 8 * NT + h) * G::O_ROW + d];
    }
    const int hh = kvh * p.rep + h0 + h;
    if (p.splits == 1) {
      static_cast<T*>(p.out)[r * p.ldo + static_cast<int64_t>(hh) * HD + d] = from_f<T>(o / total);
    } else {
      const int64_t part = (r * p.nh + hh) * p.splits + split;
      p.ws[part * HD + d] = o;
      if (d == 0) {
        float* ml = p.ws + static_cast<int64_t>(gridDim.z) * p.nh * p.splits * HD + 2 * part;
        ml[0] = top;
        ml[1] = total;
      }
    }
  }
}

bool supported(const Params& p) {
  if (p.hd != 64 && p.hd != 128 && p.hd != 256) return false;
  return p.kv.block_stride % 16 == 0 && p.kv.head_stride % 16 == 0 &&
         ((reinterpret_cast<uintptr_t>(p.kv.k) | reinterpret_cast<uintptr_t>(p.kv.v)) & 15) == 0;
}

template <typename T, int HD, int NT, bool WHOLE>
int launch_geo(Params p, int64_t B, int64_t nkv, cudaStream_t st) {
  using G = Geo<T, HD, NT, WHOLE>;
  p.groups = (p.rep + 8 * NT - 1) / (8 * NT);
  if (nkv * p.groups > 65535) return fail("fs_attention_decode_quant: too many heads");
  static bool attr[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr[dev]) {
    if (cudaFuncSetAttribute(quant_decode_tc_kernel<T, HD, NT, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             G::SMEM) != cudaSuccess)
      return check_launch("quant_decode_tc set smem");
    attr[dev] = true;
  }
  const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(nkv * p.groups), static_cast<unsigned>(B));
  launch_pdl_async(quant_decode_tc_kernel<T, HD, NT, WHOLE>, grid, 32 * WARPS, G::SMEM, st, p);
  return check_launch("quant_decode_tc_kernel");
}

template <typename T, int HD>
int launch_hd(const Params& p, int64_t B, int64_t nkv, cudaStream_t st) {
  const bool whole = p.kv.block_size % TILE == 0;
  if (p.rep > 8)   // two N tiles read the cache once for up to 16 heads
    return whole ? launch_geo<T, HD, 2, true>(p, B, nkv, st) : launch_geo<T, HD, 2, false>(p, B, nkv, st);
  return whole ? launch_geo<T, HD, 1, true>(p, B, nkv, st) : launch_geo<T, HD, 1, false>(p, B, nkv, st);
}

template <typename T>
int launch_t(const Params& p, int64_t B, int64_t nkv, cudaStream_t st) {
  return p.hd == 64 ? launch_hd<T, 64>(p, B, nkv, st)
                    : p.hd == 128 ? launch_hd<T, 128>(p, B, nkv, st) : launch_hd<T, 256>(p, B, nkv, st);
}

}  // namespace tc

// Joins the splits of a (row, head), weights exp2(m_split - m): four warps take the splits in turn, lanes the dims.
template <typename T>
__global__ void __launch_bounds__(128) quant_combine_kernel(Params p) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  constexpr int MAXD = 8;
  __shared__ float red[4], sums[4], part[4][32 * MAXD];
  const int64_t r = blockIdx.y;
  const int h = blockIdx.x, hd = p.hd, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n_vis = visible(p, r), base = (r * p.nh + h) * p.splits;
  const int used = static_cast<int>((n_vis + SPLIT_KEYS - 1) / SPLIT_KEYS);
  const float* ml = p.ws + static_cast<int64_t>(gridDim.y) * p.nh * p.splits * hd + 2 * base;
  const float* o = p.ws + base * hd;
  float top = -INFINITY;
  for (int s = threadIdx.x; s < used; s += blockDim.x) top = fmaxf(top, ml[2 * s]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  if (lane == 0) red[warp] = top;
  __syncthreads();
  top = safe_max(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
  float total = 0.f, acc[MAXD];
#pragma unroll
  for (int i = 0; i < MAXD; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int s = warp; s < used; s += 4) {
    const float2 v = *reinterpret_cast<const float2*>(ml + 2 * s);
    const float w = exp2f(v.x - top);
    total += w * v.y;
#pragma unroll
    for (int i = 0; i < MAXD; ++i)
      if (lane + 32 * i < hd) acc[i] = fmaf(w, o[static_cast<int64_t>(s) * hd + lane + 32 * i], acc[i]);
  }
  if (lane == 0) sums[warp] = total;
#pragma unroll
  for (int i = 0; i < MAXD; ++i) part[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  total = sums[0] + sums[1] + sums[2] + sums[3];
  for (int d = threadIdx.x; d < hd; d += blockDim.x)
    static_cast<T*>(p.out)[r * p.ldo + static_cast<int64_t>(h) * hd + d] =
        from_f<T>(n_vis == 0 ? 0.f : (part[0][d] + part[1][d] + part[2][d] + part[3][d]) / total);
}

template <typename T>
int launch_any(const Params& p, int64_t B, int64_t nkv, cudaStream_t st) {
  const size_t smem = (32 * (2 * p.hd + 1) + HEADS * p.hd) * sizeof(float);
  static bool attr[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr[dev]) {
    const int most = (32 * (2 * 256 + 1) + HEADS * 256) * static_cast<int>(sizeof(float));
    if (cudaFuncSetAttribute(quant_decode_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
      return check_launch("quant_decode set smem");
    attr[dev] = true;
  }
  const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(nkv * p.groups), static_cast<unsigned>(B));
  launch_pdl_async(quant_decode_kernel<T>, grid, 128, smem, st, p);
  return check_launch("quant_decode_kernel");
}

template <typename T>
int launch_t(const Params& p, int64_t B, int64_t nkv, cudaStream_t st) {
  if (tc::supported(p) ? tc::launch_t<T>(p, B, nkv, st) : launch_any<T>(p, B, nkv, st)) return -1;
  if (p.splits == 1) return 0;
  launch_pdl_async(quant_combine_kernel<T>, dim3(static_cast<unsigned>(p.nh), static_cast<unsigned>(B)), 128, 0, st, p);
  return check_launch("quant_combine_kernel");
}

}  // namespace

int64_t splits(int64_t n_slots) { return (n_slots + SPLIT_KEYS - 1) / SPLIT_KEYS; }

int64_t workspace_bytes(int64_t B, int64_t nh, int64_t hd, int64_t n_slots) {
  const int64_t s = splits(n_slots);
  return s <= 1 ? 0 : B * nh * s * (hd + 2) * static_cast<int64_t>(sizeof(float));
}

int launch(int dtype, const void* q, int64_t ldq, const KVCache& kv, const KVScales& sc, int64_t n_slots,
           const int64_t* positions, void* out, int64_t ldo, int64_t B, int64_t nh, int64_t nkv, int64_t hd, float scale,
           float* ws, cudaStream_t st) {
  Params p;
  p.q = q;
  p.ldq = ldq;
  p.kv = kv;
  p.sc = sc;
  p.n_slots = n_slots;
  p.positions = positions;
  p.out = out;
  p.ldo = ldo;
  p.nh = static_cast<int>(nh);
  p.rep = static_cast<int>(nh / nkv);
  p.hd = static_cast<int>(hd);
  p.splits = static_cast<int>(splits(n_slots));
  p.groups = (p.rep + HEADS - 1) / HEADS;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.ws = ws;
  p.err = error_word();
  if (!p.err) return -1;
  if (nkv * p.groups > 65535) return fail("fs_attention_decode_quant: too many heads");
  return dtype == F32 ? launch_t<float>(p, B, nkv, st) : launch_t<__nv_bfloat16>(p, B, nkv, st);
}

}  // namespace decode_quant
}  // namespace fs
