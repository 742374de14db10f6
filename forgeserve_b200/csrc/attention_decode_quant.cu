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

// Joins the splits of a (row, head): weights exp2(m_split - m).
template <typename T>
__global__ void __launch_bounds__(128) quant_combine_kernel(Params p) {
  pdl_trigger();
  pdl_wait();   // launched with PDL: everything below reads or writes other kernels' data
  const int64_t r = blockIdx.y;
  const int h = blockIdx.x, hd = p.hd;
  const int64_t n_vis = visible(p, r), base = (r * p.nh + h) * p.splits;
  const int used = static_cast<int>((n_vis + SPLIT_KEYS - 1) / SPLIT_KEYS);
  const float* ml = p.ws + static_cast<int64_t>(gridDim.y) * p.nh * p.splits * hd + 2 * base;
  float top = -INFINITY;
  for (int s = 0; s < used; ++s) top = fmaxf(top, ml[2 * s]);
  top = safe_max(top);
  for (int d = threadIdx.x; d < hd; d += blockDim.x) {
    float total = 0.f, o = 0.f;
    for (int s = 0; s < used; ++s) {
      const float w = exp2f(ml[2 * s] - top);
      total += w * ml[2 * s + 1];
      o += w * p.ws[(base + s) * hd + d];
    }
    static_cast<T*>(p.out)[r * p.ldo + static_cast<int64_t>(h) * hd + d] = from_f<T>(n_vis == 0 ? 0.f : o / total);
  }
}

template <typename T>
int launch_t(const Params& p, int64_t B, int64_t nkv, cudaStream_t st) {
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
  if (check_launch("quant_decode_kernel")) return -1;
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
