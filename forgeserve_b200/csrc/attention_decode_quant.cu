// Decode attention (one new query per row) over the 8-bit cache of kv_quant.cu: grouped query heads, slot s of a row
// visible iff s <= position and s < n_slots, scale 1/sqrt(hd), as attention_decode.cu over an unquantised cache.
//
// With codes kq, vq and scales ks, vs of a (slot, KV head) row:
//     s_j = (q . kq_j) ks_j scale,   p_j = exp(s_j - max s),   out = sum_j p_j vs_j vq_j / sum_j p_j
// so a scale is one factor on a score or on a probability, and the products run on the codes themselves.
// The floor is the cache's bytes: 2 (hd + 4) for each visible slot of each KV head, read once for all its query heads.
//
// A row's slots are cut into splits, a CTA's work each; quant_combine_kernel joins them. How they are cut follows from
// the row's visible slots and the KV heads alone (split_keys), so the order of a row's sums does not depend on the batch
// or on the table's width (a step gives the same bits eagerly, in a CUDA graph with a padded table, or in micro-batches).
// Workspace (fp32): sums [B][nh][splits][hd], then (max, sum) [B][nh][splits][2] in the log2 domain.
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

constexpr int UNIT_KEYS = 512;   // a split is a multiple of this (256 took 97 us on the 64 rows below, 1024 77, but
                                 // 16 us on one row of 4096 slots instead of 12)
constexpr int ONE_WAVE = 592;    // CTAs that run at once: 4 on each of 148 SMs
constexpr int HEADS = 8;         // query heads of one KV head that a CTA of the general kernel handles

// Slots a split of a row with n_vis visible slots: 512 while the row's CTAs fit one wave, so that a row alone spreads
// over the GPU; longer rows get longer splits, which join cheaper (2 rows of 131072 slots of 8 KV heads: 256 splits of
// 512 took 161 us, 51 of them in the join, 64 of 2048 125 us).
__host__ __device__ __forceinline__ int64_t split_keys(int64_t n_vis, int64_t nkv) {
  const int64_t units = (n_vis + UNIT_KEYS - 1) / UNIT_KEYS;
  const int64_t k = (units * nkv + ONE_WAVE - 1) / ONE_WAVE;
  return UNIT_KEYS * (k > 1 ? k : 1);
}

struct Params {
  const void* q;
  int64_t ldq;
  KVCache kv;
  KVScales sc;
  int64_t n_slots;
  const int64_t* positions;
  void* out;
  int64_t ldo;
  int B, nh, nkv, rep, hd, splits, groups;   // groups: CTAs a KV head, of HEADS (or 8 NT) query heads each
  bool q_vec;                        // rows of q on 16-byte boundaries
  int rows_per_block, rows_per_head, map_rows;   // of the tensor maps' hd-wide rows (WHOLE)
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

// What the tensor-core kernel below does not take (hd no multiple of 16, rows off 16 bytes): any hd <= 256 and layout, 32
// keys at a time as fp32 in shared memory; a warp owns two query heads, a lane one key of the scores and hd / 32 dims of
// the sums.
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
  const int64_t per = split_keys(n_vis, p.nkv), begin = split * per;
  const int64_t end = begin + per < n_vis ? begin + per : n_vis;
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
// hd a multiple of 16 up to 256, 16-byte rows; the kernel is built for HD = 64, 128 and 256, dims from hd on are zeros
// in shared memory (no bytes of the cache). The codes are exact in f16, so both products run as mma.sync m16n8k16 f16
// with fp32 sums and the scales never touch them; the query heads of the KV head are the N side (NT tiles of 8). A tcgen05
// product would want the codes widened in shared memory first; here they are widened in registers:
//     S^T (16 keys x 8 heads) = K (16 x hd) Q^T (hd x 8),   O^T (hd x 8 heads) += V^T (hd x 16) P^T (16 x 8)
// A contraction's index order is free as long as both operands agree, and so are the rows of O^T; they are chosen so
// that every lane's operand values are neighbouring bytes of a cache row: lane (g, t) = (lane / 4, lane % 4) takes, of
// keys g and g + 8, two 16-byte chunks of each 128 bytes for K (k_chunk), and of keys 2t, 2t+1, 2t+8, 2t+9 the chunk
// g for V (8 bytes of it at hd 64). P^T reaches the B layout by movmatrix.
//
// A warp takes STEP keys at a time, into a ring of its own; no barrier joins the warps before the end.
//   WHOLE (the block size is a multiple of 16, so a tile of 16 keys lies in one block): TMA boxes of 16 rows, swizzled
//     over 128 (hd 64: 64) bytes, under which both fragment reads above are free of bank conflicts.
//   otherwise every key is looked up by itself and each lane copies exactly the bytes it will use (cp.async).
//
// Q enters as f16 after a scale by a power of two that brings each head's largest |q| to [1, 2): exact for bf16 down to
// 2^-14 of it, off by 2^-25 of it below. fp32 queries enter as two halves (a value and its remainder times 2^11): 22
// bits. P enters in f16 (2^-11 of itself) as p_j vs_j against a running maximum of its own: P = exp2(s + log2 vs - mo),
// max(s + log2 vs) - mo between HEADROOM and HEADROOM + SLACK, so that the largest P lies near the end of f16's range.
// What lies 2^20 below the largest p vs of its warp's keys meets f16's smallest steps and is off by 2^-31 of that largest
// one. fp32 takes log2 vs as exponent and mantissa and P's remainder as a second product: 22 bits, then off by 2^-37 of
// the largest (a smaller SLACK leaves more HEADROOM: 64 rows of 2048 to 4096 slots 89.8 us against 88.3; remainders times
// 2^11, and codes by 2^-11 beside them, would end at 2^-42 and take 97.8). The sum l of the p is fp32 throughout.
// Maxima are raised only when a score exceeds them by SLACK: one vote a step instead of a reduction.
//
// 64 rows of 2176 to 4352 slots of 8 x 128 values, 32 query heads: 78 us with the join, 86 % of HBM (bf16 queries); 2
// rows of 131072: 91 us, 92 %. The copies alone, without a product, take 68 us of the first, the join 6.
namespace tc {

constexpr int WARPS = 4, TILE = 16, STEP = 32;   // a warp takes STEP keys (two tiles) at a time
constexpr int SEG = 4;         // steps whose places a warp looks up at once
constexpr float LOWEST = -3e38f;

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Orders this thread's earlier shared-memory accesses before later async-proxy (TMA) writes to the same bytes.
__device__ __forceinline__ void fence_proxy_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// BYTES (4, 8 or 16) from global to shared memory.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// The same, zeros where !ok (src is then not read, but still a valid address).
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

// log2(x), off by 2^-22 (of the value where that is more); 0 gives -infinity.
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 neighbouring values, by 16-byte loads where `vec`: two bf16 a word (8 words), or fp32 (16 words).
__device__ __forceinline__ void load16(const __nv_bfloat16* q, bool vec, uint32_t* x) {
  if (vec) {
    *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(q);
    *reinterpret_cast<uint4*>(x + 4) = *reinterpret_cast<const uint4*>(q + 8);
  } else {
    const uint16_t* u = reinterpret_cast<const uint16_t*>(q);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = u[2 * i] | static_cast<uint32_t>(u[2 * i + 1]) << 16;
  }
}
__device__ __forceinline__ void load16(const float* q, bool vec, uint32_t* x) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(x + 4 * i) = *reinterpret_cast<const uint4*>(q + 4 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(q[i]);
  }
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

template <typename T, int HD, int NT, bool WHOLE>
struct Geo {
  static constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;        // f16 terms of q and of p
  // What a score may exceed its reference maximum by, and where P lies at that maximum, in powers of two: together, with a
  // mantissa, below f16's 2^16.
  static constexpr float SLACK = PARTS == 2 ? 2.f : 8.f, HEADROOM = 14.f - SLACK;
  static constexpr int KS = HD / 16;                          // k steps of S^T, and m tiles of O^T
  static constexpr int KC = HD / 64;                          // 16-byte chunks a lane takes of a K row
  static constexpr int VB = HD / 8 < 16 ? 8 : 16;             // bytes a lane takes of a V row at once
  static constexpr int VC = HD / 8 / VB;                      // and how often
  static constexpr int BOX = HD < 128 ? 64 : 128;             // bytes of a box's row
  static constexpr int BOXES = HD / BOX;                      // boxes a row
  static constexpr int STEP_BYTES = STEP * HD;                // K (or V) of a step
  // A warp's ring is one step deep: K of the next step is on its way from the scores on, its V from the V product on.
  // At hd 128 two steps take the shared memory of a fourth CTA an SM (64 rows: 89 us against 80), four for CTAs alone on
  // an SM save 0.3 us of 11. Not tried at hd 64, where the issue slots, not the bytes on their way, are short.
  static constexpr int BUF = 2 * STEP_BYTES;                  // a warp's K, then V
  static constexpr int Q_OFF = WARPS * BUF;                   // q as B operands: [NT][PARTS][KS][32 lanes] of 8 bytes
  static constexpr int AT_OFF = Q_OFF + NT * PARTS * KS * 256;   // places: [2][values, scales][WARPS][LOOK]
  static constexpr int LOOK = SEG * (WHOLE ? 2 : STEP);
  static constexpr int BAR_OFF = AT_OFF + 2 * WARPS * LOOK * 16;   // a warp's barriers, K and V
  static constexpr int END = BAR_OFF + (WHOLE ? WARPS * 16 : 0);
  static constexpr int O_ROW = HD + 4;                        // padded: the lanes' writes spread over the banks
  static constexpr int O_BYTES = WARPS * 8 * NT * (O_ROW + 3) * 4;   // the merge: sums, (max, sum), weights
  static_assert(!WHOLE || O_BYTES <= BAR_OFF, "the merge must leave the barriers alone");
  static constexpr int SMEM = (O_BYTES > END ? O_BYTES : END) + (WHOLE ? 1024 : 0);   // boxes lie on 1024 bytes
  // CTAs an SM that the registers are held to, measured in bf16 (hd 128: 80 us on 64 rows at 4, 87 at 3; 16 heads a KV head
  // 65 at 3, 76 unbounded; hd 64, MHA 50 at 6, 55 at 4; hd 256 31 at 3, 34 unbounded). bf16 then spills up to 8 bytes a
  // thread, 136 at hd 256 with two N tiles; fp32 up to 28, at hd 256 188 with one N tile and 436 with two.
  static constexpr int CTAS = NT == 1 ? (HD == 64 ? (sizeof(T) == 2 ? 6 : 5) : HD == 128 ? 4 : 3)
                                      : (HD == 64 ? 4 : HD == 128 ? 3 : 2);
  // byte of a K (or V) step's 16-byte chunk `chunk` of row `row`
  static __device__ __forceinline__ int box_at(int row, int chunk) {
    const int tile = row >> 4, r = row & 15;
    if constexpr (BOX == 64) return tile * 16 * HD + r * 64 + ((chunk ^ ((r >> 1) & 3)) << 4);
    return tile * 16 * HD + (chunk >> 3) * 16 * 128 + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
  }
};
// The 16-byte chunk of a K row that lane t of a quad takes c-th: neighbours under the boxes' swizzle, four lanes' whole
// sectors in a lane's own copies.
template <int HD, bool WHOLE>
__device__ __forceinline__ int k_chunk(int t, int c) {
  return HD == 64 ? t : WHOLE ? (c >> 1) * 8 + 2 * t + (c & 1) : 4 * c + t;
}

struct Row {   // what a CTA works on: a row's query heads h0 .. h0 + heads - 1 of one KV head
  int64_t r, n_vis, per;
  int kvh, h0, heads;
};

// One split of a row. phase: steps that this warp's barriers have seen. False if a copy did not come in time.
template <typename T, int HD, int NT, bool WHOLE>
__device__ __forceinline__ bool decode_split(const Params& p, const CUtensorMap* tmK, const CUtensorMap* tmV,
                                             uint8_t* smem, const Row& row, int split, uint32_t phase) {
  using G = Geo<T, HD, NT, WHOLE>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, tl = lane & 3;
  const int64_t r = row.r, n_vis = row.n_vis, per = row.per, begin = split * per;
  const int kvh = row.kvh, h0 = row.h0, heads = row.heads;
  uint8_t* buf = smem + warp * G::BUF;
  uint64_t* kbar = reinterpret_cast<uint64_t*>(smem + G::BAR_OFF) + warp * 2;
  uint64_t* vbar = kbar + 1;
  const int n_keys = static_cast<int>(n_vis - begin < per ? n_vis - begin : per);
  const int n_steps = (n_keys + STEP - 1) / STEP;
  const int my_n = n_steps > warp ? (n_steps - warp + WARPS - 1) / WARPS : 0;   // steps warp, warp + WARPS, ..

  // Where the tiles (a row of the tensor map) or keys of SEG steps of this warp lie, -1 for bad blocks and past the last
  // visible key. Two segments, so that the next one is looked up while this one is in use.
  int64_t* at = reinterpret_cast<int64_t*>(smem + G::AT_OFF) + warp * G::LOOK;
  auto look_up = [&](int seg) {
    int64_t* dst = at + (seg & 1) * WARPS * G::LOOK * 2;
#pragma unroll
    for (int i = 0; i < (G::LOOK + 31) / 32; ++i) {
      const int k = lane + 32 * i;
      const int key = WHOLE ? (warp + WARPS * (seg * SEG + (k >> 1))) * STEP + (k & 1) * TILE
                            : (warp + WARPS * (seg * SEG + i)) * STEP + lane;
      if (k < G::LOOK) {
        int64_t a = -1, b = -1;
        if (key < n_keys) {
          int64_t col, in;
          split_slot(begin + key, p.kv.block_size, col, in);
          const int64_t blk = col < p.kv.table_cols ? p.kv.table[r * p.kv.table_stride + col] : -1;
          if (blk >= 0 && blk < p.kv.num_blocks) {
            a = WHOLE ? blk * p.rows_per_block + kvh * p.rows_per_head + in
                      : blk * p.kv.block_stride + kvh * p.kv.head_stride + in * p.hd;
            b = blk * p.sc.block_stride + kvh * p.sc.head_stride + in;
          } else {
            flag_error(p.err, ERR_BAD_SLOT);
          }
        }
        dst[k] = a;
        dst[WARPS * G::LOOK + k] = b;
      }
    }
    __syncwarp();
  };
  auto place = [&](int j) -> const int64_t* {   // of step j in `at`
    return at + ((j / SEG) & 1) * WARPS * G::LOOK * 2 + (j % SEG) * (G::LOOK / SEG);
  };

  const uint8_t* none = static_cast<const uint8_t*>(p.kv.k);   // a valid address for copies of nothing
  const uint64_t once = l2_policy_evict_first();   // each key is read once: leave L2 to the splits' partial sums
  // One warp's tiles of a step by TMA: rows past the map's end (bad blocks, tiles past the last key) read as zeros.
  auto load_boxes = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* bar, const int64_t* a) {
    if (lane == 0) {
      const int row0 = a[0] < 0 ? p.map_rows : static_cast<int>(a[0]);
      const int row1 = a[1] < 0 ? p.map_rows : static_cast<int>(a[1]);
      fence_proxy_async_smem();   // the warp's reads of the step that lay there come first
      mbar_arrive_expect_tx(bar, G::STEP_BYTES);
#pragma unroll
      for (int b = 0; b < G::BOXES; ++b) {
        tma_load_2d_hint(dst + b * 16 * G::BOX, map, bar, b * G::BOX, row0, once);
        tma_load_2d_hint(dst + 16 * HD + b * 16 * G::BOX, map, bar, b * G::BOX, row1, once);
      }
    }
  };
  // K of this warp's step j; V of it. The warp has read what lay there.
  auto issue_k = [&](int j) {
    const int64_t* a = place(j);
    if constexpr (WHOLE) {
      load_boxes(tmK, buf, kbar, a);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t o = a[gl + 8 * i];
        const uint8_t* src = o >= 0 ? static_cast<const uint8_t*>(p.kv.k) + o : none;
#pragma unroll
        for (int c = 0; c < G::KC; ++c) {
          const int d = k_chunk<HD, WHOLE>(tl, c) * 16;
          copy_async<16>(smem_u32(buf) + ((i * G::KC + c) * 32 + lane) * 16, d < p.hd ? src + d : none,
                         o >= 0 && d < p.hd);
        }
      }
    }
  };
  auto issue_v = [&](int j) {
    const int64_t* a = place(j);
    if constexpr (WHOLE) {
      load_boxes(tmV, buf + G::STEP_BYTES, vbar, a);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t o = a[(i >> 2) * TILE + 2 * tl + (i & 1) + 4 * (i & 2)];
        const uint8_t* src = o >= 0 ? static_cast<const uint8_t*>(p.kv.v) + o : none;
#pragma unroll
        for (int c = 0; c < G::VC; ++c) {
          const int d = c * 128 + gl * G::VB;
          copy_async<G::VB>(smem_u32(buf) + G::STEP_BYTES + ((i * G::VC + c) * 32 + lane) * G::VB,
                            d < p.hd ? src + d : none, o >= 0 && d < p.hd);
        }
      }
    }
  };
  float ks_next = 0.f, vs_next = 0.f;   // scales of key `lane` of the next step, zero where it is not visible or bad
  auto load_scales = [&](int j) {
    const int64_t* b = place(j) + WARPS * G::LOOK;
    const int64_t so = WHOLE ? b[lane >> 4] : b[lane];
    const bool ok = so >= 0 && (warp + WARPS * j) * STEP + lane < n_keys;
    const int64_t s = so + (WHOLE ? lane & 15 : 0);
    ks_next = ok ? p.sc.k[s] : 0.f;
    vs_next = ok ? p.sc.v[s] : 0.f;
  };
  auto commit = [] {
    if constexpr (!WHOLE) asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // Waits for K (V) of step j; false if it did not come within the time limit.
  auto wait = [&](uint64_t* bar, int j) -> bool {
    if constexpr (WHOLE) {
      return __all_sync(0xffffffffu, mbar_wait(bar, (phase + j) & 1, p.err));
    } else {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      return true;
    }
  };
  look_up(0);
  if (my_n > 0) load_scales(0);
  if (my_n > 0) issue_k(0);
  commit();
  if (my_n > 0) issue_v(0);
  commit();

  // Q as B operands: lane (gl, tl) holds of head 8 n + gl the dims 16 k_chunk(tl, c) + 4 i + 0..3, k step 4 c + i, after
  // the head's scale. Every warp finds the scales, and writes its share of the k steps to shared memory.
  uint2* qf = reinterpret_cast<uint2*>(smem + G::Q_OFF) + lane;
  float fs[NT][2];   // score factors of this lane's columns, heads 8 n + 2 tl and + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool real = 8 * n + gl < heads;
    const T* q = static_cast<const T*>(p.q) + r * p.ldq +
                 static_cast<int64_t>(kvh * p.rep + h0 + (real ? 8 * n + gl : 0)) * p.hd;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int WORDS = F32 ? 16 : 8;   // of 16 values
    uint32_t x[G::KC * WORDS], top = 0;
#pragma unroll
    for (int c = 0; c < G::KC; ++c) {
      const int d = k_chunk<HD, WHOLE>(tl, c) * 16;
      if (d < p.hd) {
        load16(q + d, p.q_vec, x + c * WORDS);
      } else {
#pragma unroll
        for (int i = 0; i < WORDS; ++i) x[c * WORDS + i] = 0;
      }
    }
#pragma unroll
    for (int i = 0; i < G::KC * WORDS; ++i)
      top = F32 ? max(top, x[i] & 0x7fffffffu) : __vmaxu2(top, x[i] & 0x7fff7fffu);
    if constexpr (!F32) top = max(top & 0xffff0000u, top << 16);
    if (!real) top = 0;
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^-e of the largest value as two factors, each inside fp32's range
    const int e = top < 0x00800000u ? (top ? -126 : 0) : static_cast<int>(top >> 23) - 127, e0 = e >> 1, e1 = e - e0;
    const float f0 = real ? __int_as_float((127 - e0) << 23) : 0.f, f1 = __int_as_float((127 - e1) << 23);
    const float back = p.scale_log2 * __int_as_float((127 + e0) << 23) * __int_as_float((127 + e1) << 23);
    fs[n][0] = __shfl_sync(0xffffffffu, back, 8 * tl);        // lane (2 tl, 0)
    fs[n][1] = __shfl_sync(0xffffffffu, back, 8 * tl + 4);
#pragma unroll
    for (int ks = 0; ks < G::KS; ++ks) {
      if ((ks & (WARPS - 1)) != warp) continue;
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = F32 ? x[4 * ks + i] : i & 1 ? x[2 * ks + i / 2] & 0xffff0000u : x[2 * ks + i / 2] << 16;
        y[i] = __uint_as_float(w) * f0 * f1;
      }
      const uint2 hi = make_uint2(pack_half2(y[0], y[1]), pack_half2(y[2], y[3]));
      qf[(n * G::PARTS * G::KS + ks) * 32] = hi;
      if constexpr (G::PARTS == 2) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
        qf[((n * G::PARTS + 1) * G::KS + ks) * 32] =
            make_uint2(pack_half2((y[0] - a.x) * 2048.f, (y[1] - a.y) * 2048.f),
                       pack_half2((y[2] - b.x) * 2048.f, (y[3] - b.y) * 2048.f));
      }
    }
  }
  __syncthreads();

  // This lane's columns are heads 8 n + 2 tl and + 1 of each N tile n. Maxima start below every finite score instead of at
  // -infinity, so that no difference to them is of two infinities.
  float m[NT][2], mo[NT][2], l[NT][2], acc[NT][G::KS][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[n][c] = mo[n][c] = LOWEST;
      l[n][c] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < G::KS; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
  }

  int late = 0;   // 1, 2: K, V did not come in time
  int j = 0;
  for (; j < my_n; ++j) {
    const float ks_mine = ks_next, vs_mine = vs_next;
    if (j % SEG == SEG / 2 - 1 && j + SEG / 2 + 1 < my_n) look_up(j / SEG + 1);
    if (j + 1 < my_n) load_scales(j + 1);
    if (!wait(kbar, j)) {
      late = 1;
      break;
    }
    float s[2][NT][4];   // keys 16 t + gl (c 0, 1) and + 8 (c 2, 3)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float a[NT][G::PARTS][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int q = 0; q < G::PARTS; ++q) a[n][q][0] = a[n][q][1] = a[n][q][2] = a[n][q][3] = 0.f;
#pragma unroll
      for (int c = 0; c < G::KC; ++c) {
        const int a0_at = WHOLE ? G::box_at(t * TILE + gl, k_chunk<HD, WHOLE>(tl, c)) : ((2 * t * G::KC + c) * 32 + lane) * 16;
        const int a1_at = WHOLE ? G::box_at(t * TILE + gl + 8, k_chunk<HD, WHOLE>(tl, c)) : a0_at + G::KC * 512;
        const uint4 u = *reinterpret_cast<const uint4*>(buf + a0_at);
        const uint4 w = *reinterpret_cast<const uint4*>(buf + a1_at);
        const uint32_t ku[4] = {u.x, u.y, u.z, u.w}, kw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = lo_pair(ku[i]), a1 = lo_pair(kw[i]), a2 = hi_pair(ku[i]), a3 = hi_pair(kw[i]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < G::PARTS; ++q) {
              const uint2 b = qf[((n * G::PARTS + q) * G::KS + c * 4 + i) * 32];
              mma_f16(a[n][q], a0, a1, a2, a3, b.x, b.y);
            }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[t][n][c] = a[n][0][c];
          if constexpr (G::PARTS == 2) s[t][n][c] = fmaf(a[n][1][c], 1.f / 2048.f, s[t][n][c]);
        }
    }
    __syncwarp();
    if (j + 1 < my_n) issue_k(j + 1);   // over the K just read
    commit();

    // Scores in the log2 domain; e: the exponent (fp32: its whole part) of the value's scale.
    float e_mine, mant_mine = 1.f;
    if constexpr (G::PARTS == 2)
      split_scale(vs_mine, e_mine, mant_mine);
    else
      e_mine = lg2(vs_mine);
    float e[2][2], mant[2][2];
    const int left = n_keys - (warp + WARPS * j) * STEP;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int key = t * TILE + 8 * k + gl;
        const float ks = __shfl_sync(0xffffffffu, ks_mine, key);
        e[t][k] = __shfl_sync(0xffffffffu, e_mine, key);
        if constexpr (G::PARTS == 2) mant[t][k] = __shfl_sync(0xffffffffu, mant_mine, key);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) s[t][n][2 * k + c] *= fs[n][c] * ks;
      }
    if (left < STEP) {   // keys that are not visible
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (t * TILE + 8 * (c >> 1) + gl >= left) {
#pragma unroll
            for (int n = 0; n < NT; ++n) s[t][n][c] = -INFINITY;
          }
    }
    bool raise = false;
    float tm[NT][2], tmo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        tm[n][c] = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
        tmo[n][c] = fmaxf(fmaxf(s[0][n][c] + e[0][0], s[0][n][c + 2] + e[0][1]),
                          fmaxf(s[1][n][c] + e[1][0], s[1][n][c + 2] + e[1][1]));
        raise |= tm[n][c] > m[n][c] + G::SLACK || tmo[n][c] > mo[n][c] + (G::HEADROOM + G::SLACK);
      }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = tm[n][c], y = tmo[n][c];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, o));
          }
          x = fmaxf(x, m[n][c]);
          y = fmaxf(y - G::HEADROOM, mo[n][c]);
          const float co = ex2(mo[n][c] - y);
          l[n][c] *= ex2(m[n][c] - x);
#pragma unroll
          for (int i = 0; i < G::KS; ++i) {
            acc[n][i][c] *= co;
            acc[n][i][c + 2] *= co;
          }
          m[n][c] = x;
          mo[n][c] = y;
        }
    }
    uint32_t pb[2][NT][G::PARTS][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          l[n][c & 1] += ex2(s[t][n][c] - m[n][c & 1]);
          w[c] = ex2(s[t][n][c] + e[t][c >> 1] - mo[n][c & 1]);
          if constexpr (G::PARTS == 2) w[c] *= mant[t][c >> 1];
        }
        const uint32_t p0 = pack_half2(w[0], w[1]), p1 = pack_half2(w[2], w[3]);
        pb[t][n][0][0] = movmatrix_trans(p0);
        pb[t][n][0][1] = movmatrix_trans(p1);
        if constexpr (G::PARTS == 2) {
          const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&p0));
          const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
          pb[t][n][1][0] = movmatrix_trans(pack_half2(w[0] - f0.x, w[1] - f0.y));
          pb[t][n][1][1] = movmatrix_trans(pack_half2(w[2] - f1.x, w[3] - f1.y));
        }
      }
    if (!wait(vbar, j)) {
      late = 2;
      break;
    }
    if (WHOLE && left < STEP) {   // whatever lies behind the last visible key, NaN codes too, becomes zeros
      for (int i = lane; i < (STEP - left) * (HD / 16); i += 32) {
        const int row = left + i / (HD / 16);
        *reinterpret_cast<uint4*>(buf + G::STEP_BYTES + G::box_at(row, i % (HD / 16))) =
            make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
    }
    // V: words of four dims of this lane's four keys, paired by key.
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < G::VC; ++c) {
        uint32_t v[4][G::VB / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = t * TILE + 2 * tl + (i & 1) + 4 * (i & 2);
          const int v_at = !WHOLE ? (((t * 4 + i) * G::VC + c) * 32 + lane) * G::VB
                                  : HD == 64 ? G::box_at(row, gl >> 1) + (gl & 1) * 8 : G::box_at(row, c * 8 + gl);
          const uint8_t* src = buf + G::STEP_BYTES + v_at;
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
                mma_f16(acc[n][(c * (G::VB / 4) + w) * 2 + half], a0, a1, a2, a3, pb[t][n][q][0], pb[t][n][q][1]);
          }
      }
    __syncwarp();
    if (j + 1 < my_n) issue_v(j + 1);
    commit();
  }
  if constexpr (WHOLE) {
    if (late) {   // let the copies in flight land (bounded) before the shared memory is given back or used again
      const int k = late == 1 ? j : j + 1;   // the K in flight
      if (k < my_n) mbar_wait(kbar, (phase + k) & 1, p.err);
      mbar_wait(vbar, (phase + j) & 1, p.err);
    }
  } else {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }

  // Merge the warps: sums against max m, through shared memory.
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], o);
  if (__syncthreads_or(late)) return false;   // buffers, q and offsets are free; a CTA that gave up leaves no result
  float* osm = reinterpret_cast<float*>(smem);                     // [WARPS][8 NT][O_ROW]
  float* msm = osm + WARPS * 8 * NT * G::O_ROW;                    // [WARPS][8 NT][2]
  float* wsm = msm + WARPS * 8 * NT * 2;                           // [8 NT][WARPS]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int h = warp * 8 * NT + 8 * n + 2 * tl + c;
      const float f = exp2f(0.5f * (mo[n][c] - m[n][c]));   // twice: scales near fp32's end leave its range at once
#pragma unroll
      for (int i = 0; i < G::KS; ++i)
        *reinterpret_cast<float2*>(osm + h * G::O_ROW + i / (G::VB / 2) * 128 + gl * G::VB + 2 * (i % (G::VB / 2))) =
            make_float2(acc[n][i][c] * f * f, acc[n][i][c + 2] * f * f);
      if (gl == 0) {
        msm[2 * h] = m[n][c];
        msm[2 * h + 1] = l[n][c];
      }
    }
  __syncthreads();
  const int64_t part0 = (r * p.nh + kvh * p.rep + h0) * p.splits + split;   // head h: part0 + h * splits
  for (int h = threadIdx.x; h < heads; h += blockDim.x) {
    float top = LOWEST, total = 0.f, f[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, msm[2 * (w * 8 * NT + h)]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      f[w] = ex2(msm[2 * (w * 8 * NT + h)] - top);
      total += f[w] * msm[2 * (w * 8 * NT + h) + 1];
    }
#pragma unroll
    for (int w = 0; w < WARPS; ++w) wsm[h * WARPS + w] = f[w];
    if (p.splits == 1) {
      msm[2 * h] = total;   // over warp 0's maximum, which this thread alone has read
    } else {
      float* ml = p.ws + static_cast<int64_t>(gridDim.z) * p.nh * p.splits * p.hd +
                  2 * (part0 + static_cast<int64_t>(h) * p.splits);
      ml[0] = top;
      ml[1] = total;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x * 4; i < heads * HD; i += blockDim.x * 4) {
    const int h = i / HD, d = i % HD;
    if (d >= p.hd) continue;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(osm + (w * 8 * NT + h) * G::O_ROW + d);
      const float f = wsm[h * WARPS + w];
      o.x = fmaf(f, x.x, o.x);
      o.y = fmaf(f, x.y, o.y);
      o.z = fmaf(f, x.z, o.z);
      o.w = fmaf(f, x.w, o.w);
    }
    if (p.splits == 1) {   // divided after the sum, as the join divides: a row's only split gives the same bits there
      T* dst = static_cast<T*>(p.out) + r * p.ldo + static_cast<int64_t>(kvh * p.rep + h0 + h) * p.hd + d;
      const float total = msm[2 * h];
      dst[0] = from_f<T>(o.x / total);
      dst[1] = from_f<T>(o.y / total);
      dst[2] = from_f<T>(o.z / total);
      dst[3] = from_f<T>(o.w / total);
    } else {
      *reinterpret_cast<float4*>(p.ws + (part0 + static_cast<int64_t>(h) * p.splits) * p.hd + d) = o;
    }
  }
  return true;
}

template <typename T, int HD, int NT, bool WHOLE>
__global__ void __launch_bounds__(32 * WARPS, Geo<T, HD, NT, WHOLE>::CTAS)
    quant_decode_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, Params p) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  using G = Geo<T, HD, NT, WHOLE>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = WHOLE ? reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023))
                        : smem_raw;
  Row row;
  row.r = blockIdx.z;
  row.kvh = blockIdx.y / p.groups;
  row.h0 = (blockIdx.y % p.groups) * 8 * NT;
  row.heads = p.rep - row.h0 < 8 * NT ? p.rep - row.h0 : 8 * NT;
  row.n_vis = visible(p, row.r);
  row.per = split_keys(row.n_vis, p.nkv);
  if (blockIdx.x * row.per >= row.n_vis) {   // the join does not read an empty split
    if (p.splits == 1)                       // a row that sees nothing
      for (int i = threadIdx.x; i < row.heads * p.hd; i += blockDim.x)
        static_cast<T*>(p.out)[row.r * p.ldo + static_cast<int64_t>(row.kvh * p.rep + row.h0) * p.hd + i] =
            from_f<T>(0.f);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if constexpr (WHOLE) {
    if (lane == 0) {
      uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::BAR_OFF) + warp * 2;
      mbar_init(&bars[0], 1);
      mbar_init(&bars[1], 1);
      fence_barrier_init();
    }
    __syncwarp();
  }
  // A grid that would hold many CTAs for splits that no row has (a table much wider than its rows) takes them in turn.
  uint32_t phase = 0;
  for (int split = blockIdx.x; split * row.per < row.n_vis; split += gridDim.x) {
    if (split != static_cast<int>(blockIdx.x)) {
      fence_proxy_async_smem();   // the merge's shared memory is the next split's ring
      __syncthreads();
    }
    if (!decode_split<T, HD, NT, WHOLE>(p, &tmK, &tmV, smem, row, split, phase)) return;
    const int64_t left = row.n_vis - split * row.per, keys = left < row.per ? left : row.per;
    const int steps = static_cast<int>((keys + STEP - 1) / STEP);
    phase += steps > warp ? (steps - warp + WARPS - 1) / WARPS : 0;
  }
}

bool supported(const Params& p) {
  if (p.hd % 16 || p.hd > 256) return false;
  return p.kv.block_stride % 16 == 0 && p.kv.head_stride % 16 == 0 &&
         ((reinterpret_cast<uintptr_t>(p.kv.k) | reinterpret_cast<uintptr_t>(p.kv.v)) & 15) == 0;
}

// Tensor maps see the cache as rows of hd bytes: whole rows between heads and blocks, and 31-bit row numbers.
bool whole_tiles(const Params& p) {
  if (p.kv.block_size % TILE || p.kv.block_stride % p.hd || p.kv.head_stride % p.hd) return false;
  if (p.kv.head_stride < 0 || p.kv.block_stride < 0) return false;
  return (p.kv.num_blocks - 1) * (p.kv.block_stride / p.hd) + (p.nkv - 1) * (p.kv.head_stride / p.hd) +
             p.kv.block_size <= INT32_MAX - 2 * TILE;
}

template <typename T, int HD, int NT, bool WHOLE>
int launch_geo(Params p, int64_t B, int64_t nkv, cudaStream_t st) {
  using G = Geo<T, HD, NT, WHOLE>;
  p.groups = (p.rep + 8 * NT - 1) / (8 * NT);
  if (nkv * p.groups > 65535) return fail("fs_attention_decode_quant: too many heads");
  CUtensorMap mk = {}, mv = {};
  if constexpr (WHOLE) {
    p.rows_per_block = static_cast<int>(p.kv.block_stride / p.hd);
    p.rows_per_head = static_cast<int>(p.kv.head_stride / p.hd);
    p.map_rows = static_cast<int>((p.kv.num_blocks - 1) * p.rows_per_block + (nkv - 1) * p.rows_per_head +
                                  p.kv.block_size);
    if (make_byte_map(&mk, p.kv.k, p.hd, p.map_rows, TILE) || make_byte_map(&mv, p.kv.v, p.hd, p.map_rows, TILE))
      return -1;
  }
  static bool attr[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr[dev]) {
    if (cudaFuncSetAttribute(quant_decode_tc_kernel<T, HD, NT, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             G::SMEM) != cudaSuccess)
      return check_launch("quant_decode_tc set smem");
    attr[dev] = true;
  }
  // at most 8 waves of CTAs: in a wider grid most stand for splits that no row has
  const int64_t each = (8 * ONE_WAVE + nkv * p.groups * B - 1) / (nkv * p.groups * B);
  const dim3 grid(static_cast<unsigned>(p.splits < each ? p.splits : each), static_cast<unsigned>(nkv * p.groups),
                  static_cast<unsigned>(B));
  launch_pdl_async(quant_decode_tc_kernel<T, HD, NT, WHOLE>, grid, 32 * WARPS, G::SMEM, st, mk, mv, p);
  return check_launch("quant_decode_tc_kernel");
}

template <typename T, int HD>
int launch_hd(const Params& p, int64_t B, int64_t nkv, cudaStream_t st) {
  const bool whole = whole_tiles(p);
  if (p.rep > 8)   // two N tiles read the cache once for up to 16 heads
    return whole ? launch_geo<T, HD, 2, true>(p, B, nkv, st) : launch_geo<T, HD, 2, false>(p, B, nkv, st);
  return whole ? launch_geo<T, HD, 1, true>(p, B, nkv, st) : launch_geo<T, HD, 1, false>(p, B, nkv, st);
}

template <typename T>
int launch_t(const Params& p, int64_t B, int64_t nkv, cudaStream_t st) {
  return p.hd <= 64 ? launch_hd<T, 64>(p, B, nkv, st)
                    : p.hd <= 128 ? launch_hd<T, 128>(p, B, nkv, st) : launch_hd<T, 256>(p, B, nkv, st);
}

}  // namespace tc

// Joins the splits of a (row, head), W warps (1 or 4) each: weights exp2(m_split - m), then four interleaved sums over the
// splits, joined pairwise; the order, and so the bits, are the same for both W. Four warps each while their CTAs are few,
// the loads then come at once (1024 pairs of 4 splits of hd 256: 28 us with the splits against 31); one warp each from
// 4096 pairs on (4096 pairs of 8 splits of hd 128: 63 us against 67).
constexpr int MAX_SPLITS = ONE_WAVE;
template <typename T, int W>
__global__ void __launch_bounds__(128) quant_combine_kernel(Params p) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  constexpr int TEAMS = 4 / W;
  __shared__ float weights[TEAMS][MAX_SPLITS];
  __shared__ float2 sums[4][64];   // W = 4: the warps' sums of 64 columns (pairs of dims)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = p.hd, cols = hd / 2, team = warp / W;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * TEAMS + team;
  if (id >= static_cast<int64_t>(p.B) * p.nh) return;   // W = 1: whole warps, which no barrier joins
  const int64_t r = id / p.nh, base = id * p.splits;
  const int64_t n_vis = visible(p, r), per = split_keys(n_vis, p.nkv);
  const int used = static_cast<int>((n_vis + per - 1) / per);
  const float2* ml = reinterpret_cast<const float2*>(p.ws + static_cast<int64_t>(p.B) * p.nh * p.splits * hd) + base;
  const float2* src = reinterpret_cast<const float2*>(p.ws + base * hd);
  T* dst = static_cast<T*>(p.out) + r * p.ldo + (id - r * p.nh) * hd;
  float* w = weights[team];
  // W = 4: the first splits' values are asked for before their number is known (the workspace holds p.splits of each)
  constexpr int EARLY = W == 1 ? 1 : 4;
  float2 early[EARLY][2];
  if constexpr (W == 4) {
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
      const int s = warp + 4 * i;
      early[i][0] = early[i][1] = make_float2(0.f, 0.f);
      if (s < p.splits) {
        if (lane < cols) early[i][0] = src[static_cast<int64_t>(s) * cols + lane];
        if (lane + 32 < cols) early[i][1] = src[static_cast<int64_t>(s) * cols + lane + 32];
      }
    }
  }
  const float2 first = lane < p.splits ? ml[lane] : make_float2(0.f, 0.f);
  float top = lane < used ? first.x : -INFINITY, total = 0.f;
  for (int s = lane + 32; s < used; s += 32) top = fmaxf(top, ml[s].x);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  top = safe_max(top);
  for (int s = lane; s < used; s += 32) {
    const float2 v = s < 32 ? first : ml[s];
    const float f = exp2f(v.x - top);
    total = fmaf(f, v.y, total);
    if (W == 1 || warp == 0) w[s] = f;
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) total += __shfl_xor_sync(0xffffffffu, total, i);
  if constexpr (W == 1) __syncwarp(); else __syncthreads();
  for (int c0 = 0; c0 < cols; c0 += 64) {   // two columns a lane at a time
    const int c = c0 + lane, d = c + 32;
    constexpr int SUMS = W == 1 ? 4 : 1;
    float2 a[SUMS], b[SUMS];
#pragma unroll
    for (int g = 0; g < SUMS; ++g) a[g] = b[g] = make_float2(0.f, 0.f);
    auto add = [&](int g, int s, float2 x, float2 y) {
      const float f = w[s];
      a[g].x = fmaf(f, x.x, a[g].x);
      a[g].y = fmaf(f, x.y, a[g].y);
      b[g].x = fmaf(f, y.x, b[g].x);
      b[g].y = fmaf(f, y.y, b[g].y);
    };
    auto load = [&](int s, int col) {
      return col < cols ? src[static_cast<int64_t>(s) * cols + col] : make_float2(0.f, 0.f);
    };
    int s0 = W == 1 ? 0 : warp;
    if (W == 4 && c0 == 0) {
#pragma unroll
      for (int i = 0; i < EARLY; ++i, s0 += 4)
        if (s0 < used) add(0, s0, early[i][0], early[i][1]);
    }
#pragma unroll(W == 1 ? 2 : 8)
    for (; s0 < used; s0 += 4) {
#pragma unroll
      for (int g = 0; g < SUMS; ++g)
        if (s0 + g < used) add(g, s0 + g, load(s0 + g, c), load(s0 + g, d));
    }
    if constexpr (W == 1) {
      a[0].x = (a[0].x + a[1].x) + (a[2].x + a[3].x);
      a[0].y = (a[0].y + a[1].y) + (a[2].y + a[3].y);
      b[0].x = (b[0].x + b[1].x) + (b[2].x + b[3].x);
      b[0].y = (b[0].y + b[1].y) + (b[2].y + b[3].y);
    } else {
      __syncthreads();   // the columns before these are read
      sums[warp][lane] = a[0];
      sums[warp][lane + 32] = b[0];
      __syncthreads();
      if (warp == 0) {
        a[0].x = (sums[0][lane].x + sums[1][lane].x) + (sums[2][lane].x + sums[3][lane].x);
        a[0].y = (sums[0][lane].y + sums[1][lane].y) + (sums[2][lane].y + sums[3][lane].y);
      } else if (warp == 1) {
        b[0].x = (sums[0][lane + 32].x + sums[1][lane + 32].x) + (sums[2][lane + 32].x + sums[3][lane + 32].x);
        b[0].y = (sums[0][lane + 32].y + sums[1][lane + 32].y) + (sums[2][lane + 32].y + sums[3][lane + 32].y);
      }
    }
    if ((W == 1 || warp == 0) && c < cols) {
      dst[2 * c] = from_f<T>(n_vis == 0 ? 0.f : a[0].x / total);
      dst[2 * c + 1] = from_f<T>(n_vis == 0 ? 0.f : a[0].y / total);
    }
    if ((W == 1 || warp == 1) && d < cols) {
      dst[2 * d] = from_f<T>(n_vis == 0 ? 0.f : b[0].x / total);
      dst[2 * d + 1] = from_f<T>(n_vis == 0 ? 0.f : b[0].y / total);
    }
  }
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
  const int64_t pairs = B * p.nh;
  if (pairs >= 4096)
    launch_pdl_async(quant_combine_kernel<T, 1>, static_cast<unsigned>((pairs + 3) / 4), 128, 0, st, p);
  else
    launch_pdl_async(quant_combine_kernel<T, 4>, static_cast<unsigned>(pairs), 128, 0, st, p);
  return check_launch("quant_combine_kernel");
}

}  // namespace

// Most splits that any row of up to n_slots visible slots has (split_keys): the grid and the workspace are made for it.
int64_t splits(int64_t nkv, int64_t n_slots) {
  const int64_t units = (n_slots + UNIT_KEYS - 1) / UNIT_KEYS, most = (ONE_WAVE + nkv - 1) / nkv;
  return units < most ? units : most;
}

int64_t workspace_bytes(int64_t B, int64_t nh, int64_t nkv, int64_t hd, int64_t n_slots) {
  const int64_t s = splits(nkv, n_slots);
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
  p.B = static_cast<int>(B);
  p.nh = static_cast<int>(nh);
  p.rep = static_cast<int>(nh / nkv);
  p.hd = static_cast<int>(hd);
  p.nkv = static_cast<int>(nkv);
  p.splits = static_cast<int>(splits(nkv, n_slots));
  p.groups = (p.rep + HEADS - 1) / HEADS;
  p.q_vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && ldq % (dtype == F32 ? 4 : 8) == 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.ws = ws;
  p.err = error_word();
  if (!p.err) return -1;
  if (nkv * p.groups > 65535) return fail("fs_attention_decode_quant: too many heads");
  return dtype == F32 ? launch_t<float>(p, B, nkv, st) : launch_t<__nv_bfloat16>(p, B, nkv, st);
}

}  // namespace decode_quant
}  // namespace fs
