// Verification of drafted tokens against the target's probabilities (speculative sampling), from given random numbers.
//
// For a sequence with n drafted tokens d_i, target rows p_0..p_n, draft rows q_0..q_{n-1} (without them q_i is 1 at d_i
// and 0 elsewhere) and uniforms u_0..u_K:
//   d_i is accepted when u_i q_i(d_i) < p_i(d_i); a = the first i that is not, or n;
//   w = max(p_a - q_a, 0), or p_a where that is all zero (a < n); w = p_n (a = n);
//   the next token is the first j with C_j > u_K C_V, C the running sums of w.
// A token drawn this way is distributed as the target's own. Which j that is depends on sums of up to V terms next to a
// border, so products, differences and sums are taken in 64 bits (the product and each difference of two 32-bit or
// 16-bit values are then exact or within 2^-53): in 32 bits about one row in 50 of 151936 columns would take a
// neighbouring token, and the order of the additions would show.
//
// HBM bound: the row p_a and, after a refusal, q_a are read once, and nothing else of the K + 1 rows but one value each.
// One cluster of C CTAs per sequence, each with a contiguous slice, each warp of a CTA with a contiguous part of that;
// the CTAs exchange their sums through distributed shared memory, and the one CTA whose slice holds the border reads
// one warp's part of it again (some KB, from L2), then a sixteenth of that, down to one step of a warp. So there is no
// workspace, one launch, and a fixed order of additions.
// 256 sequences of 151936 fp32 columns, each with a refused token (311 MB), take 57.5 us, 5.4 TB/s or 0.84 of the measured copy
// bandwidth; 64 of 128256 bf16 columns (31 MB) 13.9 us; one sequence 8.6 us, the latency of its chain (token,
// its probabilities, the row, the exchange, the narrowing). More CTAs than fit at once took 61 to 82 us, three CTAs an SM, which spill, 67 us and more.
#include "ckb200_verify.h"
#include "common.cuh"

#include <climits>

namespace ckb {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kPerSm = 2;  // resident CTAs of an SM: with 4 vectors of p and of q in flight a thread, 128 KB an SM

struct VerifyArgs {
  const void *target, *draft;
  const long long *tokens, *counts;
  const float* uniforms;
  long long* out;
  long long* accepted;
  long long target_batch, target_row, draft_batch, draft_row;  // strides in elements
  int drafts, vocab;
  int part;  // columns of one warp, a multiple of 32 vectors' elements
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(r));
  return r;
}
// Stores v into the same shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ void store_remote(double* p, unsigned rank, double v) {
  unsigned at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory");
}

// A probability that is NaN or negative counts as 0 (fmaxf drops a NaN), the target's and the draft's alike.
__device__ __forceinline__ float clean(float p) { return fmaxf(p, 0.0f); }
// What one element weighs: max(p - q, 0), q cleaned: a NaN or negative p is above no such q, and nothing is above an infinite one.
__device__ __forceinline__ double weight(float p, float q) { return p > q ? (double)p - (double)q : 0.0; }

// A lane's columns of one step, as they were loaded (widened only where they are used, so that several steps' loads fit
// the registers). kVec: one 16-byte vector, else one element. Columns from `end` on are zeros and weigh nothing.
template <typename T, bool kVec>
struct Piece {
  static constexpr int N = VecN<T>::N;
  static constexpr bool kCleanOnce = sizeof(T) == 4;  // by clean_all, not element by element
  uint4 r;
  __device__ __forceinline__ void load(const T* row, int i, int end) {
    r = make_uint4(0u, 0u, 0u, 0u);
    if (row != nullptr && i < end) r = ld_stream(row + i);
  }
  __device__ __forceinline__ void widen(float (&f)[N]) const { unpack16(r, f, (const T*)nullptr); }
  // Cleans K vectors of fp32. As unsigned integers, negative values and NaN are above infinity, which three-way maxima find with
  // half an instruction an element; as a rule there are none, and nothing more is done (256 sequences of
  // 151936 columns 57.5 us; with every element cleaned 59.1 us, with none 57.2 us).
  template <int K>
  static __device__ __forceinline__ void clean_all(Piece (&p)[K]) {
    unsigned most = 0u;
#pragma unroll
    for (int s = 0; s < K; ++s) most = __vimax3_u32(__vimax3_u32(most, p[s].r.x, p[s].r.y), p[s].r.z, p[s].r.w);
    if (most <= 0x7f800000u) return;
#pragma unroll
    for (int s = 0; s < K; ++s) {
      float f[N];
      p[s].widen(f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = clean(f[e]);
      p[s].r = pack16(f, (const T*)nullptr);
    }
  }
};
template <typename T>
struct Piece<T, false> {
  static constexpr int N = 1;
  static constexpr bool kCleanOnce = false;
  T v;
  __device__ __forceinline__ void load(const T* row, int i, int end) {
    v = row != nullptr && i < end ? row[i] : from_f32<T>(0.0f);
  }
  __device__ __forceinline__ void widen(float (&f)[1]) const { f[0] = to_f32(v); }
};

// A sequence's weights: p alone (q null), p - q, or p without one column.
template <typename T, bool kVec>
struct Weights {
  using Part = Piece<T, kVec>;
  static constexpr int N = Part::N;
  const T *p, *q;
  int without;  // a column that weighs nothing, or -1
  // The weights of columns i .. i + N - 1 (pq cleaned where that is done at once).
  __device__ __forceinline__ void of(const Part& pp, const Part& pq, int i, double (&w)[N]) const {
    float fp[N], fq[N];
    pp.widen(fp);
    pq.widen(fq);
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = weight(fp[e], Part::kCleanOnce ? fq[e] : clean(fq[e]));
    if ((unsigned)(without - i) < (unsigned)N) {  // asked once for all N columns
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i + e == without) w[e] = 0.0;
    }
  }
};

// The whole block's sums of [lo + warp * sub, + sub) below hi, into warp_sums.
template <typename T, bool kVec>
__device__ __forceinline__ void sum_parts(const Weights<T, kVec>& w, int lo, int hi, int sub, double* warp_sums) {
  constexpr int N = Weights<T, kVec>::N;
  constexpr int kStep = 32 * N;          // columns of a warp's step
  constexpr int kAhead = kVec ? 4 : 8;   // steps whose loads are in flight together
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int begin = (int)min((long long)lo + (long long)warp * sub, (long long)hi);
  const int end = (int)min((long long)begin + sub, (long long)hi);
  double sum = 0.0;
  for (int i = begin; i < end; i += kAhead * kStep) {
    Piece<T, kVec> pp[kAhead], pq[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      pp[s].load(w.p, i + s * kStep + lane * N, end);
      pq[s].load(w.q, i + s * kStep + lane * N, end);
    }
    if constexpr (Piece<T, kVec>::kCleanOnce) Piece<T, kVec>::clean_all(pq);
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      double some[N];
      w.of(pp[s], pq[s], i + s * kStep + lane * N, some);
#pragma unroll
      for (int e = 0; e < N; ++e) sum += some[e];
    }
  }
  sum = warp_sum<32, double>(sum);
  if (lane == 0) warp_sums[warp] = sum;
  __syncthreads();
}

// The first of n sums with which the running sum (from `base` on) passes the bound, else the last that is not zero
// (-1: none). `base` becomes the running sum before it. Every caller with the same sums finds the same one.
__device__ __forceinline__ int find_part(const double* sums, int n, double bound, double& base) {
  int found = -1;
  double run = base;
  for (int k = 0; k < n; ++k) {
    if (!(sums[k] > 0.0)) continue;
    found = k;
    base = run;
    run += sums[k];
    if (run > bound) break;
  }
  return found;
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads, kPerSm) verify_rows(const VerifyArgs a) {
  constexpr int N = kVec ? VecN<T>::N : 1;
  constexpr int kStep = 32 * N;
  __shared__ double cta_sums[2][kMaxCluster];
  __shared__ double warp_sums[kWarps];
  __shared__ int first_refused;
  cluster_arrive();  // every CTA of the cluster runs before one stores into another's memory
  pdl_wait();
  pdl_trigger();
  const int ctas = cluster_size(), rank = cluster_rank();
  const long long b = blockIdx.x / ctas;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* target = (const T*)a.target + b * a.target_batch;
  const T* draft = a.draft == nullptr ? nullptr : (const T*)a.draft + b * a.draft_batch;
  const long long* tokens = a.tokens + b * a.drafts;
  const float* uniforms = a.uniforms + b * (a.drafts + 1);

  const long long count = a.counts == nullptr ? a.drafts : a.counts[b];
  const int n = count < 0 ? 0 : count > a.drafts ? a.drafts : (int)count;
  if (warp == 0) {
    int refused = n;
    for (int first = 0; first < n; first += 32) {
      const int i = first + lane;
      bool fine = true;
      if (i < n) {
        const long long d = tokens[i];
        fine = false;
        if (d >= 0 && d < a.vocab) {
          const double q = draft == nullptr ? 1.0 : (double)clean(to_f32(draft[i * a.draft_row + d]));
          fine = (double)uniforms[i] * q < (double)to_f32(target[i * a.target_row + d]);
        }
      }
      const unsigned bad = ~__ballot_sync(0xffffffffu, fine);
      if (bad != 0u) {
        refused = first + __ffs(bad) - 1;
        break;
      }
    }
    if (lane == 0) first_refused = refused;
  }
  __syncthreads();
  const int at = first_refused;
  Weights<T, kVec> w;
  w.p = target + at * a.target_row;
  w.q = at < n && draft != nullptr ? draft + at * a.draft_row : nullptr;
  w.without = at < n && draft == nullptr ? (int)max(-1LL, min(tokens[at], (long long)a.vocab)) : -1;

  int lo = (int)min((long long)rank * kWarps * a.part, (long long)a.vocab);
  int hi = (int)min((long long)lo + (long long)kWarps * a.part, (long long)a.vocab);
  int owner = -1;
  double base = 0.0, bound = 0.0;
  // A second turn only where a refusal left no weight at all: then the target's own row is drawn from.
  for (int turn = 0; turn < 2; ++turn) {
    sum_parts(w, lo, hi, a.part, warp_sums);
    double total = 0.0;
    for (int k = 0; k < kWarps; ++k) total += warp_sums[k];
    if (turn == 0) cluster_wait();
    if (threadIdx.x < ctas) store_remote(&cta_sums[turn][rank], threadIdx.x, total);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    // Every thread of the cluster adds the same sums in the same order, so all find the same owner.
    double all = 0.0;
    for (int c = 0; c < ctas; ++c) all += cta_sums[turn][c];
    if (all > 0.0) {
      bound = (double)uniforms[a.drafts] * all;
      owner = find_part(cta_sums[turn], ctas, bound, base);
      break;
    }
    if (at >= n) break;
    w.q = nullptr;
    w.without = -1;
  }

  long long* out = a.out + b * (a.drafts + 1);
  if (rank == 0) {
    for (int i = threadIdx.x; i <= a.drafts; i += kThreads) {
      if (i != at) out[i] = i < at ? tokens[i] : -1;
      else if (owner < 0) out[i] = -1;
    }
    if (threadIdx.x == 0) a.accepted[b] = at;
  }
  if (owner != rank) return;
  // The owner narrows its slice: the warp's part that holds the border, a sixteenth of that, ... down to one step.
  int sub = a.part;
  while (true) {
    const int k = max(0, find_part(warp_sums, kWarps, bound, base));
    lo = (int)min((long long)lo + (long long)k * sub, (long long)hi);
    hi = (int)min((long long)lo + sub, (long long)hi);
    if (hi - lo <= kStep) break;
    sub = ((hi - lo + kWarps - 1) / kWarps + kStep - 1) / kStep * kStep;
    __syncthreads();  // warp_sums are read
    sum_parts(w, lo, hi, sub, warp_sums);
  }
  if (warp != 0) return;
  Piece<T, kVec> pp, pq[1];
  pp.load(w.p, lo + lane * N, hi);
  pq[0].load(w.q, lo + lane * N, hi);
  if constexpr (Piece<T, kVec>::kCleanOnce) Piece<T, kVec>::clean_all(pq);
  double mine[N], sum = 0.0;
  w.of(pp, pq[0], lo + lane * N, mine);
  int last = -1;  // this lane's last column with any weight
#pragma unroll
  for (int e = 0; e < N; ++e) {
    sum += mine[e];
    if (mine[e] > 0.0) last = lo + lane * N + e;
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += t;
  }
  double run = __shfl_up_sync(0xffffffffu, sum, 1);
  run = base + (lane == 0 ? 0.0 : run);
  int hit = -1;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    run += mine[e];
    if (hit < 0 && mine[e] > 0.0 && run > bound) hit = lo + lane * N + e;
  }
  const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, last >= 0);
  if (hits != 0u) hit = __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
  else if (some != 0u) hit = __shfl_sync(0xffffffffu, last, 31 - __clz(some));  // the sums' rounding hid the border
  if (lane == 0) out[at] = hit;
}

template <typename T, bool kVec>
int start(VerifyArgs a, long long batch, cudaStream_t stream) {
  constexpr int kStep = 32 * (kVec ? VecN<T>::N : 1);
  const int sms = device_sm_count();
  // The most CTAs for a sequence with which the batch still fits the GPU at once, while each warp keeps a step of its own.
  int ctas = kMaxCluster;
  while (ctas > 1 && (batch * ctas > (long long)kPerSm * sms || (long long)(ctas - 1) * kWarps * kStep >= a.vocab)) ctas /= 2;
  const long long warps = (long long)ctas * kWarps;
  const long long part = (a.vocab + warps - 1) / warps;
  a.part = (int)((part + kStep - 1) / kStep * kStep);
  if (batch * ctas > INT_MAX) return -1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CKB_PDL ? 2 : 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, verify_rows<T, kVec>, a);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return (int)err;
  }
  return (int)cudaGetLastError();
}

template <typename T>
int dispatch(const VerifyArgs& a, long long batch, cudaStream_t stream) {
  constexpr int N = VecN<T>::N;
  const bool vec = a.vocab % N == 0 && aligned16(a.target) && a.target_batch % N == 0 && a.target_row % N == 0 &&
                   (a.draft == nullptr || (aligned16(a.draft) && a.draft_batch % N == 0 && a.draft_row % N == 0));
  return vec ? start<T, true>(a, batch, stream) : start<T, false>(a, batch, stream);
}

}  // namespace
}  // namespace ckb

using namespace ckb;

CKB_EXPORT int ckb_verify_launch(const void* target, const void* draft, const void* tokens, const void* counts,
                                 const float* uniforms, void* out, void* accepted, long long target_batch,
                                 long long target_row, long long draft_batch, long long draft_row, long long batch,
                                 int drafts, int vocab, int dtype, cudaStream_t stream) {
  if (batch <= 0) return 0;
  if (batch > INT_MAX || drafts < 0 || drafts >= (1 << 20) || vocab < 1 || vocab > (1 << 30) || target == nullptr || uniforms == nullptr ||
      out == nullptr || accepted == nullptr || (drafts > 0 && tokens == nullptr))
    return -1;
  const VerifyArgs a{target, drafts == 0 ? nullptr : draft, (const long long*)tokens, (const long long*)counts, uniforms,
                     (long long*)out, (long long*)accepted, target_batch, target_row, draft_batch, draft_row, drafts,
                     vocab, 0};
  if (dtype == kF32) return dispatch<float>(a, batch, stream);
  if (dtype == kBF16) return dispatch<__nv_bfloat16>(a, batch, stream);
  return -1;
}
