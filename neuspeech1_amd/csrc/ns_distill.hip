// Distillation over logits that exist: the student's loss and gradient (ns_distill_topk) and the teacher's lists (ns_topk_logits).
//
//   loss_i = (1 - alpha) (lse(z_i) - z_i[label_i]) + alpha T^2 sum_k p_ik (log p_ik - (z_i[idx_ik] / T - lse(z_i / T))),   p_i = softmax(top_i / T)
//   dz_i   = g [ w1 softmax(z_i) + w2 softmax(z_i / T) - w1 onehot(label_i) - w2 sum_k p_ik onehot(idx_ik) ],   w1 = 1 - alpha, w2 = alpha T
//
// Both are bound by the one read of the logits (and the one write of their gradient): a workgroup takes a row, 16 B per lane and access, and
// keeps it in REGISTERS between the statistics and what needs them (V = 51 865 at 16 bits: 7 accesses, 28 registers of 1024 threads), so
// every logit crosses HBM once.  Rows longer than that are read again (from the 4-MiB L2 of the XCD, mostly).
// Rows may start at any element: the accesses of a row begin at its first 16-B boundary, its ragged ends are element accesses.
#include "ns_common.h"

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int DT_MAX_K = 256;

template <class E> struct vec { static constexpr int N = 16 / (int)sizeof(E); typedef E t __attribute__((ext_vector_type(16 / sizeof(E)))); };

// A row's elements as 16-B chunks: chunk c holds the elements [c N - sh, (c + 1) N - sh); the first and the last one may be ragged.
template <class E, int NC, int NT>
struct row_view {
  typedef typename vec<E>::t V;
  static constexpr int N = vec<E>::N;
  const E* p;
  int n, sh, chunks;
  V reg[NC > 0 ? NC : 1];
  __device__ __forceinline__ void init(const E* row, int len) {
    p = row; n = len;
    sh = (int)(((size_t)row & 15) / sizeof(E));
    chunks = (n + sh + N - 1) / N;
  }
  __device__ __forceinline__ V fetch(int c) const {
    const int j = c * N - sh;
    V v;
    if (j >= 0 && j + N <= n) {
      v = *(const V*)(p + j);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = j + e >= 0 && j + e < n ? p[j + e] : (E)(-INFINITY);
    }
    return v;
  }
  __device__ __forceinline__ void load() {
    if (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = threadIdx.x + i * NT;
        if (c < chunks) reg[i] = fetch(c);
        else {
#pragma unroll
          for (int e = 0; e < N; ++e) reg[i][e] = (E)(-INFINITY);
        }
      }
    }
  }
  // f(first element index of the chunk, chunk); elements outside the row are -inf
  template <class F> __device__ __forceinline__ void each(F f) const {
    if (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = threadIdx.x + i * NT;
        if (c < chunks) f(c * N - sh, reg[i]);
      }
    } else {
      for (int c = threadIdx.x; c < chunks; c += NT) f(c * N - sh, fetch(c));
    }
  }
};

template <int NT> __device__ __forceinline__ float block_max(float v, float* sh) {
  v = ns_wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) v = fmaxf(v, sh[i]);
  return v;
}
template <int NT> __device__ __forceinline__ float block_sum(float v, float* sh) {
  v = ns_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) v += sh[i];
  return v;
}
template <int NT> __device__ __forceinline__ int block_count(int v, int* sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) v += sh[i];
  return v;
}

// ------------------------------------------------------------------------------------------------ the student
__global__ __launch_bounds__(1024) void dt_count_kernel(const int64_t* __restrict__ labels, int rows, int V, int* __restrict__ nvalid) {
  __shared__ int sh[16];
  int c = 0;
  if (labels)
    for (int i = threadIdx.x; i < rows; i += 1024) c += labels[i] >= 0 && labels[i] < V;
  c = block_count<1024>(c, sh);
  if (threadIdx.x == 0) *nvalid = labels ? c : rows;
}

__global__ __launch_bounds__(1024) void dt_mean_kernel(const float* __restrict__ row_loss, int rows, const int* __restrict__ nvalid, float* __restrict__ loss) {
  __shared__ float sh[16];
  float s = 0.f;
  for (int i = threadIdx.x; i < rows; i += 1024) s += row_loss[i];
  s = block_sum<1024>(s, sh);
  if (threadIdx.x == 0) *loss = s / (float)max(*nvalid, 1);
}

struct DistillArgs {
  const void* z; int64_t ldz;
  const int64_t* labels; const float* tv; const int32_t* ti; int64_t ldt;
  int V, k, dual, soft_only;
  float T, w1, w2, kd;
  float* row_loss; void* dz; int64_t lddz;
  const int* nvalid; const float* loss_scale;
};

template <class E, int NC, int NT>
__global__ __launch_bounds__(NT) void distill_kernel(const DistillArgs p) {
  __shared__ float sh[16];
  __shared__ int sidx[DT_MAX_K + 1];
  __shared__ float sp[DT_MAX_K], sz[DT_MAX_K + 1];
  typedef row_view<E, NC, NT> RV;
  const int row = blockIdx.x, tid = threadIdx.x;
  const int64_t lab64 = p.labels ? p.labels[row] : -1;
  const bool has = lab64 >= 0 && lab64 < p.V;
  E* const out = p.dz ? (E*)p.dz + row * p.lddz : nullptr;
  RV r;
  r.init((const E*)p.z + row * p.ldz, p.V);
  const bool same = out && (((size_t)out ^ (size_t)r.p) & 15) == 0;
  auto put = [&](int j, typename RV::V v) __attribute__((always_inline)) {
    if (same && j >= 0 && j + RV::N <= p.V) {
      *(typename RV::V*)(out + j) = v;
    } else {
#pragma unroll
      for (int e = 0; e < RV::N; ++e)
        if (j + e >= 0 && j + e < p.V) out[j + e] = v[e];
    }
  };
  if (p.labels && !has) {                  // an ignored row: never read, zero gradient
    if (tid == 0) p.row_loss[row] = 0.f;
    if (out) {
      typename RV::V zero;
#pragma unroll
      for (int e = 0; e < RV::N; ++e) zero[e] = (E)0.f;
      for (int c = tid; c < r.chunks; c += NT) put(c * RV::N - r.sh, zero);
    }
    return;
  }
  r.load();
  // the lists: token, teacher logit / T, the student's logit there (read before any gradient overwrites it: dz may be z itself)
  for (int e = tid; e <= p.k; e += NT) {
    const int t = e == p.k ? (has ? (int)lab64 : -1) : p.ti[row * p.ldt + e];
    const bool ok = t >= 0 && t < p.V;
    sidx[e] = ok ? t : -1;
    sz[e] = ok ? (float)r.p[t] : 0.f;
    if (e < p.k) sp[e] = ok ? p.tv[row * p.ldt + e] / p.T : -INFINITY;
  }
  const float c1 = p.soft_only ? LOG2E / p.T : LOG2E, c2 = LOG2E / p.T;
  float mx = -INFINITY;
  r.each([&](int j, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < RV::N; ++e) mx = fmaxf(mx, (float)v[e]);
  });
  mx = block_max<NT>(mx, sh);
  float s1 = 0.f, s2 = 0.f;
  r.each([&](int j, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < RV::N; ++e) {
      const float x = (float)v[e] - mx;
      s1 += __builtin_amdgcn_exp2f(x * c1);
      if (p.dual) s2 += __builtin_amdgcn_exp2f(x * c2);
    }
  });
  s1 = block_sum<NT>(s1, sh);
  if (p.dual) s2 = block_sum<NT>(s2, sh);
  // the teacher's distribution and the row's loss
  float tm = -INFINITY;
  for (int e = tid; e < p.k; e += NT) tm = fmaxf(tm, sp[e]);
  tm = block_max<NT>(tm, sh);
  const bool soft = tm > -INFINITY;        // a list that names no token leaves the hard label alone
  float ts = 0.f;
  for (int e = tid; e < p.k; e += NT) ts += soft ? expf(sp[e] - tm) : 0.f;
  ts = block_sum<NT>(ts, sh);
  const float lt = logf(ts), its = 1.f / ts, lq = mx / p.T + logf(p.dual ? s2 : s1);
  float kl = 0.f;
  for (int e = tid; e < p.k; e += NT) {
    const float lp = sp[e] - tm;
    const float pr = soft ? expf(lp) * its : 0.f;
    if (pr > 0.f) kl += pr * ((lp - lt) - (sz[e] / p.T - lq));
    sp[e] = pr;
  }
  kl = block_sum<NT>(kl, sh);              // (also: every sp[] is final)
  if (tid == 0) {
    float loss = soft ? p.kd * kl : 0.f;
    if (!p.soft_only) loss += p.w1 * ((mx - sz[p.k]) + logf(s1));
    p.row_loss[row] = loss;
  }
  if (!out) return;
  const float gs = (p.loss_scale ? *p.loss_scale : 1.f) / (float)max(*p.nvalid, 1);
  const float w2 = soft ? p.w2 : 0.f;
  const float f1 = (p.dual ? p.w1 : (p.soft_only ? 0.f : p.w1) + w2) / s1, f2 = p.dual ? w2 / s2 : 0.f;
  __syncthreads();                         // sz[] has been read from z by everyone who reads it; dz may be z itself
  auto grad = [&](float z) __attribute__((always_inline)) {
    float g = f1 * __builtin_amdgcn_exp2f((z - mx) * c1);
    if (p.dual) g += f2 * __builtin_amdgcn_exp2f((z - mx) * c2);
    return g;
  };
  r.each([&](int j, typename RV::V v) __attribute__((always_inline)) {
    typename RV::V o;
#pragma unroll
    for (int e = 0; e < RV::N; ++e) o[e] = (E)(grad((float)v[e]) * gs);
    put(j, o);
  });
  // the sparse cells, each token once whatever number of entries name it, behind the dense stores
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int e = tid; e <= p.k; e += NT) {
    const int t = sidx[e];
    if (t < 0) continue;
    float q = 0.f;
    bool first = true;
    for (int o = 0; o < p.k; ++o)
      if (sidx[o] == t) { q += sp[o]; first = first && o >= e; }
    if (!first) continue;
    float g = grad(sz[e]) - w2 * q;
    if (has && t == (int)lab64) g -= p.w1;
    out[t] = (E)(g * gs);
  }
}

// ------------------------------------------------------------------------------------------------ the teacher
// The k largest of a row: (1) every thread's largest element; (2) the k-th largest of those, rounded down to its 16 leading bits, is a bound
// that at least k elements reach and, unless many elements are equal or one thread's chunks hold many of the largest, not many more; (3) the elements that
// reach it are collected and ordered by (value, lowest token first).  If more than CAP reach it, the k-th largest value itself is found bit by bit, then
// the token below which enough elements EQUAL to it lie: exactly k elements remain.  A NaN ranks above +inf.
template <class E> __device__ __forceinline__ uint32_t order_key(E x) {
  const float f = (float)x + 0.f;                             // -0 ranks as +0
  const uint32_t u = __float_as_uint(f);
  if (f != f) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <class E, int NC, int NT>
__global__ __launch_bounds__(NT) void topk_row_kernel(const E* __restrict__ z, int64_t ldz, int V, int k, float* __restrict__ vals, int32_t* __restrict__ idx,
                                                      int64_t ldo, float* __restrict__ lse) {
  constexpr int CAP = 2048;
  __shared__ uint64_t cand[CAP];
  __shared__ int shi[16];
  __shared__ float sh[16];
  __shared__ int count;
  typedef row_view<E, NC, NT> RV;
  const int row = blockIdx.x, tid = threadIdx.x;
  RV r;
  r.init(z + row * ldz, V);
  r.load();
  uint32_t best = 0;                                          // below every element's key
  float mx = -INFINITY;
  r.each([&](int j, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < RV::N; ++e)
      if (j + e >= 0 && j + e < V) { mx = fmaxf(mx, (float)v[e]); best = max(best, order_key(v[e])); }
  });
  if (lse) {
    const float m = block_max<NT>(mx, sh);
    float s = 0.f;
    const float ms = fabsf(m) == INFINITY ? 0.f : m;          // (an infinite maximum is the answer: the sum becomes 0 or infinite)
    r.each([&](int j, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < RV::N; ++e) s += __builtin_amdgcn_exp2f(((float)v[e] - ms) * LOG2E);
    });
    s = block_sum<NT>(s, sh);
    if (tid == 0) lse[row] = ms + logf(s);
  }
  // (2) the bound: leading 16 bits of the k-th largest thread maximum (0, i.e. everything, when fewer threads hold elements)
  uint32_t bound = 0;
  for (int b = 31; b >= 16; --b) {
    const uint32_t t = bound | (1u << b);
    if (block_count<NT>(best >= t, shi) >= k) bound = t;
  }
  if (tid == 0) count = 0;
  __syncthreads();
  auto collect = [&](auto take) __attribute__((always_inline)) {
    r.each([&](int j, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < RV::N; ++e) {
        if (j + e < 0 || j + e >= V) continue;
        const uint32_t key = order_key(v[e]);
        if (!take(key, j + e)) continue;
        const int at = atomicAdd(&count, 1);
        if (at < CAP) cand[at] = ((uint64_t)key << 32) | (uint32_t)~(j + e);
      }
    });
  };
  collect([&](uint32_t key, int) { return key >= bound; });
  __syncthreads();
  int n = count;
  if (n > CAP) {
    auto reach = [&](auto take) __attribute__((always_inline)) {
      int c = 0;
      r.each([&](int j, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < RV::N; ++e)
          if (j + e >= 0 && j + e < V) c += take(order_key(v[e]), j + e);
      });
      return block_count<NT>(c, shi);
    };
    uint32_t kth = 0;
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = kth | (1u << b);
      if (reach([&](uint32_t key, int) { return key >= t; }) >= k) kth = t;
    }
    const int more = reach([&](uint32_t key, int) { return key > kth; });
    int upto = 0;                                             // the largest bound below which fewer than k - more equal elements lie
    for (int b = 30; b >= 0; --b) {
      const int t = upto | (1 << b);
      if (reach([&](uint32_t key, int at) { return key == kth && at < t; }) < k - more) upto = t;
    }
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    collect([&](uint32_t key, int at) { return key > kth || (key == kth && at <= upto); });
    __syncthreads();
    n = count;
  }
  // (3) each candidate's place is the number of candidates above it
  for (int c = tid; c < n; c += NT) {
    const uint64_t me = cand[c];
    int above = 0;
    for (int o = 0; o < n; ++o) above += cand[o] > me;
    if (above < k) {
      const int t = (int)~(uint32_t)me;
      vals[row * ldo + above] = (float)r.p[t];
      idx[row * ldo + above] = t;
    }
  }
}

template <class E, template <class, int, int> class Launch, class... A>
void by_length(int V, A... a) {
  // threads and registers by the row's length: one access per thread up to 256 accesses, then 1024 threads with as many as the row needs
  const int chunks = V / vec<E>::N + 2;
  constexpr int F = sizeof(E) == 4 ? 2 : 1;      // an access holds half as many fp32 elements: twice the accesses cover the same rows
  if (chunks <= 256) Launch<E, 1, 256>::go(a...);
  else if (chunks <= 512) Launch<E, 2, 256>::go(a...);
  else if (chunks <= 1024 * 2) Launch<E, 2, 1024>::go(a...);
  else if (chunks <= 1024 * 4 * F) Launch<E, 4 * F, 1024>::go(a...);
  else if (chunks <= 1024 * 8 * F) Launch<E, 8 * F, 1024>::go(a...);
  else Launch<E, 0, 1024>::go(a...);
}

template <class E, int NC, int NT> struct distill_go {
  static void go(const DistillArgs& a, int rows, hipStream_t st) { hipLaunchKernelGGL((distill_kernel<E, NC, NT>), dim3(rows), dim3(NT), 0, st, a); }
};
template <class E, int NC, int NT> struct topk_go {
  static void go(const ns_topk_desc* d, hipStream_t st) {
    hipLaunchKernelGGL((topk_row_kernel<E, NC, NT>), dim3(d->rows), dim3(NT), 0, st, (const E*)d->logits, d->ldz, d->vocab, d->k, d->vals, d->idx, d->ldo, d->lse);
  }
};

bool elem_aligned(const void* q, int dtype) { return ((size_t)q & (dtype == NS_F32 ? 3 : 1)) == 0; }

}  // namespace

extern "C" int ns_distill_topk(const ns_distill_desc* d, void* stream) {
  NS_CHECK_ARG(d, "ns_distill_topk: null descriptor");
  NS_CHECK_ARG(d->loss_dev && d->nvalid_dev && (d->rows == 0 || (d->logits && d->row_loss && d->top_vals && d->top_idx)), "ns_distill_topk: null pointer");
  NS_CHECK_ARG(d->rows >= 0 && d->vocab > 0 && d->vocab <= (1 << 30) && d->k > 0 && d->k <= DT_MAX_K, "ns_distill_topk: bad sizes rows=%d vocab=%d k=%d (k <= %d)", d->rows,
               d->vocab, d->k, DT_MAX_K);
  NS_CHECK_ARG(d->dtype == NS_F16 || d->dtype == NS_BF16 || d->dtype == NS_F32, "ns_distill_topk: dtype %d", d->dtype);
  NS_CHECK_ARG(d->rows <= 1 || (d->ldz >= d->vocab && d->ld_top >= d->k && (!d->dlogits || d->lddz >= d->vocab)), "ns_distill_topk: row strides shorter than the rows");
  NS_CHECK_ARG(elem_aligned(d->logits, d->dtype) && elem_aligned(d->dlogits, d->dtype), "ns_distill_topk: logits not aligned to their elements");
  NS_CHECK_ARG(d->temperature >= 1e-3f && d->temperature <= 1e3f && d->alpha > 0.f && d->alpha <= 1.f, "ns_distill_topk: temperature %g in [1e-3, 1e3], alpha %g in (0, 1]",
               (double)d->temperature, (double)d->alpha);
  NS_CHECK_ARG(d->labels || d->alpha == 1.f || d->rows == 0, "ns_distill_topk: alpha %g < 1 needs labels", (double)d->alpha);
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(dt_count_kernel, dim3(1), dim3(1024), 0, st, d->labels, d->rows, d->vocab, d->nvalid_dev);
  if (d->rows > 0) {
    DistillArgs a = {};
    a.z = d->logits; a.ldz = d->ldz; a.labels = d->labels; a.tv = d->top_vals; a.ti = d->top_idx; a.ldt = d->ld_top; a.V = d->vocab; a.k = d->k;
    a.soft_only = d->alpha == 1.f;
    a.dual = !a.soft_only && d->temperature != 1.f;
    a.T = d->temperature; a.w1 = 1.f - d->alpha; a.w2 = d->alpha * d->temperature; a.kd = d->alpha * d->temperature * d->temperature;
    a.row_loss = d->row_loss; a.dz = d->dlogits; a.lddz = d->lddz; a.nvalid = d->nvalid_dev; a.loss_scale = d->loss_scale_dev;
    if (d->dtype == NS_F16) by_length<half_t, distill_go>(d->vocab, a, d->rows, st);
    else if (d->dtype == NS_BF16) by_length<__bf16, distill_go>(d->vocab, a, d->rows, st);
    else by_length<float, distill_go>(d->vocab, a, d->rows, st);
  }
  hipLaunchKernelGGL(dt_mean_kernel, dim3(1), dim3(1024), 0, st, d->row_loss, d->rows, d->nvalid_dev, d->loss_dev);
  NS_CHECK_LAUNCH("ns_distill_topk");
  return NS_OK;
}

extern "C" int ns_topk_logits(const ns_topk_desc* d, void* stream) {
  NS_CHECK_ARG(d, "ns_topk_logits: null descriptor");
  NS_CHECK_ARG(d->rows == 0 || (d->logits && d->vals && d->idx), "ns_topk_logits: null pointer");
  NS_CHECK_ARG(d->rows >= 0 && d->vocab > 0 && d->vocab <= (1 << 30) && d->k > 0 && d->k <= DT_MAX_K && d->k <= d->vocab,
               "ns_topk_logits: bad sizes rows=%d vocab=%d k=%d (k <= vocab, k <= %d)", d->rows, d->vocab, d->k, DT_MAX_K);
  NS_CHECK_ARG(d->dtype == NS_F16 || d->dtype == NS_BF16 || d->dtype == NS_F32, "ns_topk_logits: dtype %d", d->dtype);
  NS_CHECK_ARG(d->rows <= 1 || (d->ldz >= d->vocab && d->ldo >= d->k), "ns_topk_logits: row strides shorter than the rows");
  NS_CHECK_ARG(elem_aligned(d->logits, d->dtype), "ns_topk_logits: logits not aligned to their elements");
  if (d->rows == 0) return NS_OK;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == NS_F16) by_length<half_t, topk_go>(d->vocab, d, st);
  else if (d->dtype == NS_BF16) by_length<__bf16, topk_go>(d->vocab, d, st);
  else by_length<float, topk_go>(d->vocab, d, st);
  NS_CHECK_LAUNCH("ns_topk_logits");
  return NS_OK;
}
