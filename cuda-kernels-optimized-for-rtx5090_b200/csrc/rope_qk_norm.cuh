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
// is a G-wide shuffle and nothing goes through shared memory. As in rope_tokens a thread keeps up to kNormHeads heads'
// loads in flight and uses one fetch of its cos/sin values for all of them.
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

#ifndef CKB_QK_NORM_HEADS
#define CKB_QK_NORM_HEADS 5
#endif
constexpr int kNormHeads = CKB_QK_NORM_HEADS;

// Block (G, R, Z): lane threadIdx.x of heads threadIdx.y, + R, + 2R, ... of token blockIdx.x * Z + threadIdx.z. Heads
// run over q, then k, then (with a cache) v. Every thread takes every round, so a group's shuffles always meet.
template <typename T, bool kCache>
__global__ void __launch_bounds__(256) qk_norm_rope_tokens(const NormArgs a) {
  pdl_wait();
  pdl_trigger();
  const unsigned token = blockIdx.x * blockDim.z + threadIdx.z;
  const int half = a.head_dim >> 1;
  const int c = threadIdx.x * 8;
  const bool active = token < a.tokens && c < half;
  const unsigned b = token / a.seq, s = token - b * a.seq;
  const int R = blockDim.y;
  const int qk_heads = a.q_heads + a.kv_heads;
  const int heads = qk_heads + (a.slots != nullptr ? a.kv_heads : 0);
  const int G = blockDim.x;
  const unsigned lane = (threadIdx.x + G * (threadIdx.y + R * threadIdx.z)) & 31u;
  const unsigned group_mask = (G == 32 ? 0xffffffffu : ((1u << G) - 1u)) << (lane & ~(G - 1u));
  const T* q = (const T*)a.q + b * a.vq.batch + s * a.vq.token + c;
  const T* k = (const T*)a.k + b * a.vk.batch + s * a.vk.token + c;
  const T* v = (const T*)a.v + b * a.vv.batch + s * a.vv.token + c;

  const T tag{};  // selects the overloads of unpack16 / pack16
  float c1[8], s1[8], c2[8], s2[8];
  long long slot = -1;
  for (int h0 = 0; h0 < heads; h0 += kNormHeads * R) {
    uint4 ra[kNormHeads], rb[kNormHeads];
#pragma unroll
    for (int j = 0; j < kNormHeads; ++j) {  // every load of the round before any use
      const int h = h0 + threadIdx.y + j * R;
      const T* p = h < a.q_heads ? q + h * a.vq.head
                   : h < qk_heads ? k + (h - a.q_heads) * a.vk.head
                                  : v + (h - qk_heads) * a.vv.head;
      if (active && h < heads) {
        ra[j] = ld_inplace(p);
        rb[j] = ld_inplace(p + half);
      } else {
        ra[j] = rb[j] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    if (h0 == 0 && active) {  // behind the first round's loads
      const long long pos = __ldg(a.ids + token);
      slot = cache_slot(a, token);
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
    }
#pragma unroll
    for (int j = 0; j < kNormHeads; ++j) {
      const int h = h0 + threadIdx.y + j * R;
      float x[8], z[8];
      unpack16(ra[j], x, &tag);
      unpack16(rb[j], z, &tag);
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], fmaf(z[e], z[e], ss));
      for (int o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(group_mask, ss, o);
      if (!active || h >= heads) continue;
      if (h >= qk_heads) {  // v: as it is, into its cache row
        if (slot >= 0) {
          T* dst = (T*)a.value_cache + (slot * a.kv_heads + (h - qk_heads)) * a.head_dim + c;
          st_stream(dst, ra[j]);
          st_stream(dst + half, rb[j]);
        }
        continue;
      }
      const float inv = rsqrtf(ss / (float)a.head_dim + a.eps);
      const bool is_q = h < a.q_heads;
      float w1[8], w2[8];
      ld8_any(is_q ? a.q_weight : a.k_weight, a.w_dtype, c, w1);
      ld8_any(is_q ? a.q_weight : a.k_weight, a.w_dtype, c + half, w2);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float lo = x[e] * inv * w1[e], hi = z[e] * inv * w2[e];
        x[e] = lo * c1[e] - hi * s1[e];
        z[e] = hi * c2[e] + lo * s2[e];
      }
      const uint4 px = pack16(x, &tag), pz = pack16(z, &tag);
      if (is_q) {
        T* dst = (T*)a.q_out + b * a.vq_out.batch + s * a.vq_out.token + h * a.vq_out.head + c;
        st_stream(dst, px);
        st_stream(dst + half, pz);
        continue;
      }
      const int hk = h - a.q_heads;
      if (a.k_out != nullptr) {
        T* dst = (T*)a.k_out + b * a.vk_out.batch + s * a.vk_out.token + hk * a.vk_out.head + c;
        st_stream(dst, px);
        st_stream(dst + half, pz);
      }
      if (slot >= 0) {
        T* dst = (T*)a.key_cache + (slot * a.kv_heads + hk) * a.head_dim + c;
        st_stream(dst, px);
        st_stream(dst + half, pz);
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
    int lanes = 1;
    while (lanes * 16 < a.head_dim) lanes *= 2;
    const int most = 256 / lanes;  // groups of a block
    // Heads per thread: kNormHeads where that still leaves two blocks for each SM, else fewer.
    int per = kNormHeads;
    while (per > 1 && (long long)a.tokens * ((heads + per - 1) / per) < 2LL * device_sm_count() * most) --per;
    int r = (heads + per - 1) / per;
    if (r > most) r = most;
    int z = most / r;
    if (z > 64) z = 64;
    const unsigned grid = (a.tokens + z - 1) / z;
    launch_pdl(qk_norm_rope_tokens<T, kCache>, dim3(grid), dim3(lanes, r, z), 0, stream, a);
  } else {
    launch_pdl(qk_norm_rope_scalar<T, kCache>, dim3(a.tokens), dim3(32, heads < 16 ? heads : 16), 0, stream, a);
  }
  return (int)cudaGetLastError();
}

}  // namespace
}  // namespace ckb
