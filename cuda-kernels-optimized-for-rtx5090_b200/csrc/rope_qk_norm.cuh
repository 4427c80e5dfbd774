// RMSNorm of every query and key head with the rotation in the same pass, and, where asked, the paged-cache write of
// the normed, rotated keys and the values (included by rope.cu, whose load helpers it uses).
//
// For a head x of D elements with weight w (q_weight or k_weight), h = D / 2 and the token's cos/sin row:
//   y         = x * rsqrt(sum(x^2) / D + eps) * w
//   out[i]     = y[i]     * cos[i]     - y[i + h] * sin[i]
//   out[i + h] = y[i + h] * cos[i + h] + y[i]     * sin[i + h]
// all in fp32 with one rounding to the q/k dtype at the end (a separate norm kernel would round y once more, and read
// and write q and k twice).
//
// HBM bound: each element is read once and written once; cos/sin rows and weights are L2/L1 hits. A head belongs to a
// group of G = 2^n >= D / 16 lanes of one warp, lane c holding the pairs 8c..8c+7 (both halves), so the sum of squares
// is a G-wide shuffle and nothing goes through shared memory. A group takes up to kNormGroup heads of ONE kind (query, key
// or value) of a token, so it has one weight, and w cos and w sin are multiplied once for all its heads; the loads of
// kNormHeads heads are in flight all along, each replaced as soon as its head is worked on. Arithmetic is in pairs (packed
// fp32). 8 x 4096 tokens of 32 + 8 heads x 128 in bf16 take 128 us, 5.3 TB/s or 0.82 of the measured copy bandwidth (with theta
// 134 us, with the cache write 173 us). (Groups
// of mixed kinds with the weight and the angles apart took 167 us; lanes that left early, which makes every shuffle of the
// others ask who is there, 162 us.)
#pragma once

namespace ckb {
namespace {

// Offsets of a [batch, seq, heads, D] view whose last dim is contiguous, in elements.
struct View {
  long long batch, token, head;
};

struct NormArgs {
  const void *q, *k, *v, *q_weight, *k_weight, *cos_rows, *sin_rows;
  const float* inv_freq;
  const long long *ids, *slots;
  void *q_out, *k_out, *key_cache, *value_cache;
  View vq, vk, vv, vq_out, vk_out;
  long long positions, cache_slots;  // rows of the cos/sin cache; rows of the key and value caches
  unsigned tokens, seq;  // tokens = batch * seq <= INT_MAX
  int q_heads, kv_heads, head_dim, w_dtype, cache_dtype;
  float eps;
};

// 8 consecutive values of a run-time dtype as fp32 (16-byte aligned). The branch is the same for the whole grid.
__device__ __forceinline__ void ld8_any(const void* p, int dtype, long long i, float (&v)[8]) {
  if (dtype == kF32) ld8((const float*)p, i, v);
  else if (dtype == kBF16) ld8((const __nv_bfloat16*)p, i, v);
  else ld8((const __half*)p, i, v);
}
__device__ __forceinline__ float ld1_any(const void* p, int dtype, long long i) {
  if (dtype == kF32) return ((const float*)p)[i];
  if (dtype == kBF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}

// A position outside the cos/sin cache takes its first or last row, a slot outside the key and value caches is a padding
// token's: bad ids never become an address (two compares per token).
__device__ __forceinline__ long long cos_row(long long pos, long long positions) {
  return pos < 0 ? 0 : pos < positions ? pos : positions - 1;
}
__device__ __forceinline__ long long cache_slot(const NormArgs& a, unsigned token) {
  if (a.slots == nullptr) return -1;
  const long long slot = __ldg(a.slots + token);
  return slot < a.cache_slots ? slot : -1;
}

// Measured at 8 x 4096 tokens of 32 + 8 heads x 128 in bf16: 4 heads in flight of groups of 8 on two CTAs an SM (128 registers,
// 24 bytes of them spilled but for fp16 with theta) 128 us; 2 heads 140 us; 5 to 8 heads 148 us and more; groups of 4 153 us, of 16 133 us; three CTAs, which spill, 190 us.
constexpr int kNormHeads = 4;  // heads of a group whose loads are in flight
constexpr int kNormGroup = 8;  // heads of a group at most

__device__ __forceinline__ float2 as2(const float (&f)[8], int i) { return make_float2(f[2 * i], f[2 * i + 1]); }
__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// Groups of G lanes lie one after the other through the grid: group_count of a token (its queries, then keys, then, with a
// cache, values, `per` heads each), then the next token's. No lane leaves early, so the shuffles take the whole warp.
template <typename T, bool kCache>
__global__ void __launch_bounds__(256, 2) qk_norm_rope_tokens(const NormArgs a, int lanes_log, int per,
                                                                               int group_count) {
  pdl_wait();
  pdl_trigger();
  const int G = 1 << lanes_log;
  const unsigned id = blockIdx.x * (256u >> lanes_log) + (threadIdx.x >> lanes_log);
  const unsigned token = id / group_count;
  int group = id - token * group_count;
  const int half = a.head_dim >> 1;
  const int c = (threadIdx.x & (G - 1)) * 8;
  const int q_groups = (a.q_heads + per - 1) / per, k_groups = (a.kv_heads + per - 1) / per;
  const bool is_q = group < q_groups, is_v = group >= q_groups + k_groups;
  group -= is_q ? 0 : is_v ? q_groups + k_groups : q_groups;
  const int h0 = group * per;
  const bool active = token < a.tokens && c < half;
  const int count = active ? min(per, (is_q ? a.q_heads : a.kv_heads) - h0) : 0;
  const unsigned b = token / a.seq, s = token - b * a.seq;
  const long long in_head = is_q ? a.vq.head : is_v ? a.vv.head : a.vk.head;
  const T* x = (const T*)(is_q ? a.q : is_v ? a.v : a.k) + h0 * in_head + c +
               b * (is_q ? a.vq.batch : is_v ? a.vv.batch : a.vk.batch) +
               s * (is_q ? a.vq.token : is_v ? a.vv.token : a.vk.token);

  const T tag{};  // selects the overloads of unpack16 / pack16
  uint4 ra[kNormHeads], rb[kNormHeads];
  const auto fetch = [&](int j, int h) {
    ra[j] = rb[j] = make_uint4(0u, 0u, 0u, 0u);
    if (h < count) {
      ra[j] = ld_inplace(x + h * in_head);
      rb[j] = ld_inplace(x + h * in_head + half);
    }
  };
#pragma unroll
  for (int j = 0; j < kNormHeads; ++j) fetch(j, j);  // before the angles and weights
  const long long slot = is_q || token >= a.tokens ? -1 : cache_slot(a, token);
  const long long out_head = is_q ? a.vq_out.head : a.vk_out.head;
  T* out = (T*)(is_q ? a.q_out : is_v ? nullptr : a.k_out);
  if (out != nullptr)
    out += h0 * out_head + c + b * (is_q ? a.vq_out.batch : a.vk_out.batch) + s * (is_q ? a.vq_out.token : a.vk_out.token);
  T* cache = slot < 0 ? nullptr : (T*)(is_v ? a.value_cache : a.key_cache) + (slot * a.kv_heads + h0) * a.head_dim + c;
  // out_lo = x_lo inv (w_lo cos_lo) - x_hi inv (w_hi sin_lo), out_hi = x_hi inv (w_hi cos_hi) + x_lo inv (w_lo sin_hi)
  float2 lo_lo[4], lo_hi[4], hi_hi[4], hi_lo[4];
  if (active && !is_v) {
    const long long pos = __ldg(a.ids + token);
    float w1[8], w2[8], c1[8], s1[8], c2[8], s2[8];
    const void* w = is_q ? a.q_weight : a.k_weight;
    ld8_any(w, a.w_dtype, c, w1);
    ld8_any(w, a.w_dtype, c + half, w2);
    if constexpr (kCache) {
      const long long row = cos_row(pos, a.positions) * a.head_dim + c;
      ld8_any(a.cos_rows, a.cache_dtype, row, c1);
      ld8_any(a.sin_rows, a.cache_dtype, row, s1);
      ld8_any(a.cos_rows, a.cache_dtype, row + half, c2);
      ld8_any(a.sin_rows, a.cache_dtype, row + half, s2);
    } else {
      const float p = (float)pos;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sincosf(p * __ldg(a.inv_freq + c + e), &s1[e], &c1[e]);
        c2[e] = c1[e];
        s2[e] = s1[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo_lo[e] = __fmul2_rn(as2(w1, e), as2(c1, e));
      lo_hi[e] = __fmul2_rn(as2(w2, e), make_float2(-s1[2 * e], -s1[2 * e + 1]));
      hi_hi[e] = __fmul2_rn(as2(w2, e), as2(c2, e));
      hi_lo[e] = __fmul2_rn(as2(w1, e), as2(s2, e));
    }
  }
  for (int first = 0; first < per; first += kNormHeads) {
#pragma unroll
    for (int j = 0; j < kNormHeads; ++j) {
      const int h = first + j;
      float f[8], g[8];
      unpack16(ra[j], f, &tag);
      unpack16(rb[j], g, &tag);
      uint4 px = ra[j], pz = rb[j];
      fetch(j, h + kNormHeads);
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = __ffma2_rn(as2(f, e), as2(f, e), __ffma2_rn(as2(g, e), as2(g, e), sum));
      float ss = sum.x + sum.y;
      for (int o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (h >= count) continue;
      if (!is_v) {  // a value goes to its cache row as it is
        const float2 inv = twice(rsqrtf(ss / (float)a.head_dim + a.eps));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 lo = __fmul2_rn(as2(f, e), inv), hi = __fmul2_rn(as2(g, e), inv);
          const float2 u = __ffma2_rn(lo, lo_lo[e], __fmul2_rn(hi, lo_hi[e]));
          const float2 v = __ffma2_rn(hi, hi_hi[e], __fmul2_rn(lo, hi_lo[e]));
          f[2 * e] = u.x;
          f[2 * e + 1] = u.y;
          g[2 * e] = v.x;
          g[2 * e + 1] = v.y;
        }
        px = pack16(f, &tag);
        pz = pack16(g, &tag);
      }
      if (out != nullptr) {
        st_stream(out + h * out_head, px);
        st_stream(out + h * out_head + half, pz);
      }
      if (cache != nullptr) {
        st_stream(cache + h * a.head_dim, px);
        st_stream(cache + h * a.head_dim + half, pz);
      }
    }
  }
}

// Any even D, alignment and strides: a warp per head, block (32, R) per token, each head read twice (the second time
// from L1). A lane reads and writes only its own elements, so in place holds here too.
template <typename T, bool kCache>
__global__ void __launch_bounds__(512) qk_norm_rope_scalar(const NormArgs a) {
  pdl_wait();
  pdl_trigger();
  const unsigned token = blockIdx.x;
  const unsigned b = token / a.seq, s = token - b * a.seq;
  const int half = a.head_dim >> 1;
  const int qk_heads = a.q_heads + a.kv_heads;
  const int heads = qk_heads + (a.slots != nullptr ? a.kv_heads : 0);
  const long long pos = a.ids[token];
  const long long slot = cache_slot(a, token);
  for (int h = threadIdx.y; h < heads; h += blockDim.y) {
    if (h >= qk_heads) {
      if (slot >= 0) {
        const T* p = (const T*)a.v + b * a.vv.batch + s * a.vv.token + (h - qk_heads) * a.vv.head;
        T* dst = (T*)a.value_cache + (slot * a.kv_heads + (h - qk_heads)) * a.head_dim;
        for (int i = threadIdx.x; i < a.head_dim; i += 32) dst[i] = p[i];
      }
      continue;
    }
    const bool is_q = h < a.q_heads;
    const int hh = is_q ? h : h - a.q_heads;
    const View& vi = is_q ? a.vq : a.vk;
    const View& vo = is_q ? a.vq_out : a.vk_out;
    const T* p = (const T*)(is_q ? a.q : a.k) + b * vi.batch + s * vi.token + hh * vi.head;
    T* out = (T*)(is_q ? a.q_out : a.k_out);
    if (out != nullptr) out += b * vo.batch + s * vo.token + hh * vo.head;
    T* cache = is_q || slot < 0 ? nullptr : (T*)a.key_cache + (slot * a.kv_heads + hh) * a.head_dim;
    const void* w = is_q ? a.q_weight : a.k_weight;
    float ss = 0.0f;
    for (int i = threadIdx.x; i < half; i += 32) {
      const float x = to_f32(p[i]), z = to_f32(p[i + half]);
      ss = fmaf(x, x, fmaf(z, z, ss));
    }
    const float inv = rsqrtf(warp_sum(ss) / (float)a.head_dim + a.eps);
    for (int i = threadIdx.x; i < half; i += 32) {
      float c1, s1, c2, s2;
      if constexpr (kCache) {
        const long long row = cos_row(pos, a.positions) * a.head_dim + i;
        c1 = ld1_any(a.cos_rows, a.cache_dtype, row);
        s1 = ld1_any(a.sin_rows, a.cache_dtype, row);
        c2 = ld1_any(a.cos_rows, a.cache_dtype, row + half);
        s2 = ld1_any(a.sin_rows, a.cache_dtype, row + half);
      } else {
        sincosf((float)pos * a.inv_freq[i], &s1, &c1);
        c2 = c1;
        s2 = s1;
      }
      const float lo = to_f32(p[i]) * inv * ld1_any(w, a.w_dtype, i);
      const float hi = to_f32(p[i + half]) * inv * ld1_any(w, a.w_dtype, i + half);
      const T x = from_f32<T>(lo * c1 - hi * s1), z = from_f32<T>(hi * c2 + lo * s2);
      if (out != nullptr) {
        out[i] = x;
        out[i + half] = z;
      }
      if (cache != nullptr) {
        cache[i] = x;
        cache[i + half] = z;
      }
    }
  }
}

inline bool vector_view(const void* p, const View& v) {
  return aligned16(p) && v.batch % 8 == 0 && v.token % 8 == 0 && v.head % 8 == 0;
}

template <typename T, bool kCache>
int start_qk_norm(const NormArgs& a, cudaStream_t stream) {
  const int heads = a.q_heads + a.kv_heads + (a.slots != nullptr ? a.kv_heads : 0);
  const bool vec = a.head_dim % 16 == 0 && a.head_dim <= 512 && vector_view(a.q, a.vq) && vector_view(a.k, a.vk) &&
                   vector_view(a.q_out, a.vq_out) && (a.k_out == nullptr || vector_view(a.k_out, a.vk_out)) &&
                   (a.slots == nullptr || (vector_view(a.v, a.vv) && aligned16(a.key_cache) &&
                                           aligned16(a.value_cache))) &&
                   aligned16(a.q_weight) && aligned16(a.k_weight) &&
                   (kCache ? aligned16(a.cos_rows) && aligned16(a.sin_rows) : aligned16(a.inv_freq));
  if (vec) {
    int lanes_log = 0;
    while (16 << lanes_log < a.head_dim) ++lanes_log;
    const int most = 256 >> lanes_log;  // groups of a block
    // Heads per group: the most that still leaves two blocks for each SM.
    int per = kNormGroup, groups = 0;
    while (true) {
      groups = (a.q_heads + per - 1) / per + (a.slots != nullptr ? 2 : 1) * ((a.kv_heads + per - 1) / per);
      if (per == 1 || (long long)a.tokens * groups >= 2LL * device_sm_count() * most) break;
      per /= 2;
    }
    const long long all = (long long)a.tokens * groups;
    if (all > UINT_MAX - 256) return -1;
    launch_pdl(qk_norm_rope_tokens<T, kCache>, dim3((unsigned)((all + most - 1) / most)), dim3(256), 0, stream, a, lanes_log,
               per, groups);
  } else {
    launch_pdl(qk_norm_rope_scalar<T, kCache>, dim3(a.tokens), dim3(32, heads < 16 ? heads : 16), 0, stream, a);
  }
  return (int)cudaGetLastError();
}

}  // namespace
}  // namespace ckb
