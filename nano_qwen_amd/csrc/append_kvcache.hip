// Appending keys and values to a paged cache of e4m3 codes with a scale for each
// block of tokens and head (gfx950), with the q/k RMS norm and the rotary
// embedding on the way.  No counterpart in the reference, whose cache holds the
// model's own type (layers/attention.py:10-40).
//
// A block is `unit` tokens of a page (32, 64, 128 or 256); token t of the cache
// row of block c = slot / unit and head h stands for code * scale[c, h].
//
// Mathematics, per row x of one head, in fp32:
//   y = x / sqrt(mean(x^2) + eps) * (w + weight_offset)      (with weights)
//   z = y with its first R dims rotated by cos_sin[pos]        (R > 0)
// rounded once to the tensor's type (q_out, k_out).  The rows of a call that fall
// into one block of one head are a run.  With amax their largest finite |z|,
//   e = the smallest exponent in [-60, 60] with amax <= 448 * 2^e
//   s = 2^e if the run holds the block's first token, else max(s_old, 2^e)
// and the codes are e4m3(z / s) (nearest even, saturating; NaN stays NaN).  Where
// s grew, the codes of the block's tokens before the run become
// e4m3(code * s_old / s): with powers of two that only moves exponents, exactly,
// but for codes that end below 2^-6.  e4m3's precision is relative, so a finer
// scale than a power of two would gain nothing but the range's last factor of 2.
#include <algorithm>

#include "nq_device.hpp"

namespace nq {
namespace {

constexpr int kThreads = 256;
constexpr int kMinExp = -60, kMaxExp = 60;  // of a scale: products with it stay far inside fp32

struct AppendArgs {
  const uint8_t *q;
  int64_t q_row, q_head;  // strides in bytes
  const uint8_t *k, *v;
  int64_t k_row, v_row;
  const int64_t *positions;
  const float *cos_sin;  // [max_position, rot]: rot / 2 cosines, then rot / 2 sines
  int64_t max_position;
  int rot;
  const uint8_t *q_w, *k_w;  // null: no norm
  float eps, w_off;
  uint8_t *q_out;
  int64_t qo_row, qo_head;
  uint8_t *k_out;  // null: the keys are stored as they come
  int64_t ko_row;
  uint8_t *k_cache, *v_cache;
  float *k_scale, *v_scale;  // [num_slots / unit, hkv]
  const int32_t *slots;
  int64_t num_slots;
  int unit, n, hq, hkv;
  int chunk, run_wgs;  // rows whose runs a workgroup takes, and workgroups of runs
};

template <class T>
__device__ inline void row8(const uint8_t *p, float (&x)[8]) {
  const u32x4 w = load16(p);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    x[2 * t] = T::to_float(static_cast<uint16_t>(w[t] & 0xffffu));
    x[2 * t + 1] = T::to_float(static_cast<uint16_t>(w[t] >> 16));
  }
}
template <class T>
__device__ inline void store8(uint8_t *p, const float (&x)[8]) {
  const u32x4 w{T::pack2(x[0], x[1]), T::pack2(x[2], x[3]), T::pack2(x[4], x[5]), T::pack2(x[6], x[7])};
  __builtin_nontemporal_store(w, reinterpret_cast<u32x4 *>(p));
}

// Row of one head, 8 dims in each of LPU adjacent lanes (lane l of them): normed
// and rotated.  The rotary partner of dim e, e +- rot / 2, is rot / 16 lanes away.
template <class T, int LPU>
__device__ inline void transform(const AppendArgs &a, const uint8_t *weight, int64_t pos, float (&x)[8]) {
  constexpr int D = 8 * LPU;
  const int lane = threadIdx.x & 63, e0 = 8 * (threadIdx.x % LPU);
  if (weight) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int off = LPU / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, LPU);
    const float r = 1.0f / __builtin_sqrtf(ss * (1.0f / D) + a.eps);
    float w[8];
    row8<T>(weight + 2 * e0, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * (w[i] + a.w_off);
  }
  if (a.rot > 0) {
    const int half = a.rot >> 1;
    const bool rotates = e0 < a.rot, first = e0 < half;
    const int partner = rotates ? (first ? lane + (half >> 3) : lane - (half >> 3)) : lane;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], partner, 64);
    const bool bad = pos < 0 || pos >= a.max_position;
    if (rotates) {
      const float *cs = a.cos_sin + (bad ? 0 : pos) * a.rot + (first ? e0 : e0 - half);
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const f32x4 c = *reinterpret_cast<const f32x4 *>(cs + i), s = *reinterpret_cast<const f32x4 *>(cs + half + i);
#pragma unroll
        for (int t = 0; t < 4; ++t) x[i + t] = x[i + t] * c[t] + y[i + t] * (first ? -s[t] : s[t]);
      }
    }
    if (bad) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
    }
  }
}

__device__ inline float block_scale(float amax) {
  const uint32_t b = f2u(amax);
  const int e = static_cast<int>(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);  // 448 = 1.75 * 2^8
  return u2f(static_cast<uint32_t>(min(max(e, kMinExp), kMaxExp) + 127) << 23);
}

// Largest finite |x| so far.
__device__ inline float finite_max(float m, const float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = __builtin_fabsf(x[i]);
    m = v < __builtin_huge_valf() ? fmaxf(m, v) : m;
  }
  return m;
}

// Eight codes times f, coded again.
__device__ inline u32x2 recode(const u32x2 &c, float f) {
  u32x2 r;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int w = static_cast<int>(c[t]);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    r[t] = fp8x4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
  }
  return r;
}

// Workgroups 0 .. run_wgs - 1 (with a cache): the runs that start in rows chunk * i .. of one
// head, of K or of V.  The others: the query rows of one token each.
template <class T, int LPU>
__global__ __launch_bounds__(kThreads) void append_kernel(const AppendArgs a) {
  constexpr int D = 8 * LPU, RPP = kThreads / LPU;  // rows per pass of the workgroup
  const int lane = threadIdx.x & 63, l = threadIdx.x % LPU, r0 = threadIdx.x / LPU;
  if (static_cast<int>(blockIdx.x) >= a.run_wgs) {
    const int64_t tok = static_cast<int>(blockIdx.x) - a.run_wgs;
    const int64_t pos = a.rot > 0 ? a.positions[tok] : 0;
    for (int h = r0; h < a.hq; h += RPP) {
      float x[8];
      row8<T>(a.q + tok * a.q_row + h * a.q_head + 16 * l, x);
      transform<T, LPU>(a, a.q_w, pos, x);
      store8<T>(a.q_out + tok * a.qo_row + h * a.qo_head + 16 * l, x);
    }
    if (!a.k_cache)  // no runs: the keys are these workgroups' too
      for (int h = r0; h < a.hkv; h += RPP) {
        float x[8];
        row8<T>(a.k + tok * a.k_row + (h * D + 8 * l) * 2, x);
        transform<T, LPU>(a, a.k_w, pos, x);
        store8<T>(a.k_out + tok * a.ko_row + (h * D + 8 * l) * 2, x);
      }
    return;
  }
  __shared__ float lds_max[kThreads / 64];
  const int heads = 2 * a.hkv, hw = blockIdx.x % heads, i = blockIdx.x / heads;
  const bool is_v = hw >= a.hkv;
  const int h = is_v ? hw - a.hkv : hw;
  const uint8_t *src = (is_v ? a.v : a.k) + h * D * 2 + 16 * l;
  const int64_t src_row = is_v ? a.v_row : a.k_row;
  uint8_t *cache = is_v ? a.v_cache : a.k_cache;
  float *scales = is_v ? a.v_scale : a.k_scale;
  // rows of the chunk that begin a run
  const int row = i * a.chunk + lane;
  bool begins = false;
  if (lane < a.chunk && row < a.n) {
    const int32_t s = a.slots[row];
    const bool stored = s >= 0 && s < a.num_slots;
    begins = !stored || row == 0 || s % a.unit == 0 || a.slots[row - 1] != s - 1;
  }
  uint64_t todo = __builtin_amdgcn_ballot_w64(begins);
  while (todo != 0) {
    const int r = i * a.chunk + static_cast<int>(__builtin_ctzll(todo));
    todo &= todo - 1;
    const int32_t slot = __builtin_amdgcn_readfirstlane(a.slots[r]);
    const bool stored = slot >= 0 && slot < a.num_slots;
    const int off = stored ? slot % a.unit : 0;
    int len = 1;
    if (stored) {
      const int most = min(a.unit - off, a.n - r);
      for (int b = 0; b < most; b += 64) {
        const bool stop = b + lane >= most || a.slots[r + b + lane] != slot + b + lane;
        const uint64_t m = __builtin_amdgcn_ballot_w64(stop);
        len = b + (m ? static_cast<int>(__builtin_ctzll(m)) : 64);
        if (m) break;
      }
    }
    auto value = [&](int t, float (&x)[8]) {
      row8<T>(src + (r + t) * src_row, x);
      if (!is_v) transform<T, LPU>(a, a.k_w, a.rot > 0 ? a.positions[r + t] : 0, x);
    };
    float amax = 0.f;
    for (int t = r0; t < len; t += RPP) {
      float x[8];
      value(t, x);
      if (!is_v && a.k_out) store8<T>(a.k_out + (r + t) * a.ko_row + h * D * 2 + 16 * l, x);
      amax = finite_max(amax, x);
    }
    if (!stored) continue;  // the whole workgroup
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    const int64_t c = slot / a.unit * static_cast<int64_t>(a.hkv) + h;
    const float was = off > 0 ? scales[c] : 0.f;
    __syncthreads();  // the last run's maxima have been read
    if (lane == 0) lds_max[threadIdx.x / 64] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) amax = fmaxf(amax, lds_max[w]);
    const float need = block_scale(amax);
    const float s = off > 0 ? fminf(fmaxf(was, need), u2f((kMaxExp + 127u) << 23)) : need;
    const float inv = 1.0f / s;
    if (threadIdx.x == 0 && s != was) scales[c] = s;
    uint8_t *dst = cache + (static_cast<int64_t>(slot - off) * a.hkv + h) * D + 8 * l;
    if (off > 0 && s > was) {
      for (int t = r0; t < off; t += RPP) {
        u32x2 *p = reinterpret_cast<u32x2 *>(dst + static_cast<int64_t>(t) * a.hkv * D);
        *p = recode(*p, was * inv);
      }
    }
    for (int t = r0; t < len; t += RPP) {
      float x[8];
      value(t, x);
      *reinterpret_cast<u32x2 *>(dst + static_cast<int64_t>(off + t) * a.hkv * D) =
          u32x2{fp8x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv), fp8x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv)};
    }
  }
}

template <class T>
void launch(const AppendArgs &a, int head_dim, unsigned grid, hipStream_t s) {
  if (head_dim == 128)
    append_kernel<T, 16><<<grid, kThreads, 0, s>>>(a);
  else
    append_kernel<T, 32><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_append_kvcache(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k,
                                 int64_t k_row_stride, const void *v, int64_t v_row_stride, const int64_t *positions,
                                 const float *cos_sin_cache, int64_t max_position, int rotary_dim,
                                 const void *q_weight, const void *k_weight, float eps, float weight_offset,
                                 void *q_out, int64_t q_out_row_stride, int64_t q_out_head_stride, void *k_out,
                                 int64_t k_out_row_stride, void *k_cache, void *v_cache, float *k_scale,
                                 float *v_scale, const int32_t *slot_mapping, int64_t num_slots, int scale_block,
                                 int64_t num_tokens, int num_q_heads, int num_kv_heads, int head_dim, int dtype,
                                 void *stream) {
  const char *what = "append_kvcache";
  if (num_tokens < 0 || num_tokens > (1 << 24) || num_q_heads < 0 || num_kv_heads <= 0 || num_q_heads > 4096 ||
      num_kv_heads > 4096 || max_position < 0 || num_slots < 0)
    return fail(NQ_EINVAL, "%s: bad sizes (tokens=%lld q_heads=%d kv_heads=%d)", what, (long long)num_tokens, num_q_heads,
                num_kv_heads);
  if (head_dim != 128 && head_dim != 256)
    return fail(NQ_EUNSUPPORTED, "%s: head_dim %d (built: 128, 256)", what, head_dim);
  if (dtype != NQ_BF16 && dtype != NQ_F16) return fail(NQ_EUNSUPPORTED, "%s: dtype %d (need f16/bf16)", what, dtype);
  if (k_cache && scale_block != 32 && scale_block != 64 && scale_block != 128 && scale_block != 256)
    return fail(NQ_EUNSUPPORTED, "%s: blocks of %d tokens (built: 32, 64, 128, 256)", what, scale_block);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 16 != 0)
    return fail(NQ_EUNSUPPORTED, "%s: rotary_dim %d must be a multiple of 16 in [0, %d]", what, rotary_dim, head_dim);
  if (k_cache && (num_slots % scale_block != 0 || num_slots > 0x7fffffff))
    return fail(NQ_EINVAL, "%s: %lld slots in blocks of %d", what, (long long)num_slots, scale_block);
  if (num_tokens == 0) return NQ_OK;
  if (!k || (k_cache ? !v || !v_cache || !k_scale || !v_scale || !slot_mapping : !k_out) || (q && (!q_out || num_q_heads == 0)) ||
      (rotary_dim > 0 && (!positions || !cos_sin_cache)))
    return fail(NQ_EINVAL, "%s: null pointer", what);
  const int64_t row = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (k_row_stride < row || (k_cache && v_row_stride < row) || (k_out && k_out_row_stride < row))
    return fail(NQ_EINVAL, "%s: rows narrower than their heads", what);
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(q_out, 16) || !aligned(k_out, 16) ||
      !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(cos_sin_cache, 16) || !aligned(k_cache, 16) ||
      !aligned(v_cache, 16) || q_row_stride % 8 || q_head_stride % 8 || k_row_stride % 8 || v_row_stride % 8 ||
      q_out_row_stride % 8 || q_out_head_stride % 8 || k_out_row_stride % 8)
    return fail(NQ_EINVAL, "%s: pointers and strides must be 16-byte aligned", what);
  AppendArgs a{};
  a.q = static_cast<const uint8_t *>(q);
  a.q_row = q_row_stride * 2;
  a.q_head = q_head_stride * 2;
  a.k = static_cast<const uint8_t *>(k);
  a.v = static_cast<const uint8_t *>(v);
  a.k_row = k_row_stride * 2;
  a.v_row = v_row_stride * 2;
  a.positions = positions;
  a.cos_sin = cos_sin_cache;
  a.max_position = max_position;
  a.rot = rotary_dim;
  a.q_w = static_cast<const uint8_t *>(q_weight);
  a.k_w = static_cast<const uint8_t *>(k_weight);
  a.eps = eps;
  a.w_off = weight_offset;
  a.q_out = static_cast<uint8_t *>(q_out);
  a.qo_row = q_out_row_stride * 2;
  a.qo_head = q_out_head_stride * 2;
  a.k_out = static_cast<uint8_t *>(k_out);
  a.ko_row = k_out_row_stride * 2;
  a.k_cache = static_cast<uint8_t *>(k_cache);
  a.v_cache = static_cast<uint8_t *>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.slots = slot_mapping;
  a.num_slots = num_slots;
  a.unit = scale_block;
  a.n = static_cast<int>(num_tokens);
  a.hq = num_q_heads;
  a.hkv = num_kv_heads;
  // Rows per workgroup of runs: few rows are a decode step's, every one a run of
  // its own; of many, most continue the row before them.
  a.chunk = static_cast<int>(std::min<int64_t>(64, std::max<int64_t>(1, num_tokens / 512)));
  const int64_t runs = k_cache ? (num_tokens + a.chunk - 1) / a.chunk * 2 * num_kv_heads : 0;
  const int64_t grid = runs + (q || !k_cache ? num_tokens : 0);
  if (grid > 0x7fffffff) return fail(NQ_EINVAL, "%s: %lld tokens of %d heads", what, (long long)num_tokens, num_kv_heads);
  a.run_wgs = static_cast<int>(runs);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == NQ_BF16)
    launch<BF16>(a, head_dim, static_cast<unsigned>(grid), s);
  else
    launch<F16>(a, head_dim, static_cast<unsigned>(grid), s);
  return check_launch(what);
}
