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

template <class E> struct half_of { typedef E t; };
template <> struct half_of<float> { typedef half_t t; };
template <class E> using half_or = typename half_of<E>::t;      // (fp32 does not use it)

// A row as 16-B chunks from its first 16-B boundary, plus at most one element per thread from its ragged ends: threads 0 .. take the elements before
// the boundary, threads 64 .. those behind the last whole chunk (extra_j: this thread's, or -1).
template <class E, int NC, int NT>
struct row_view {
  typedef typename vec<E>::t V;
  static constexpr int N = vec<E>::N;
  const E* p;
  const ns_u4v* body;
  int head, chunks, extra_j;
  float extra;
  ns_u4v reg[NC > 0 ? NC : 1];
  __device__ __forceinline__ void init(const E* row, int n) {
    p = row;
    head = min(n, (int)((0 - (size_t)row) & 15) / (int)sizeof(E));
    chunks = (n - head) / N;
    body = (const ns_u4v*)(row + head);
    const int tail = n - head - chunks * N, t = threadIdx.x;
    extra_j = t < head ? t : (t >= 64 && t - 64 < tail ? head + chunks * N + t - 64 : -1);
    extra = -INFINITY;
  }
  // STREAM: nothing reads the row again (with its stores marked alike: 228 -> 204 us for 4096 bf16 rows of 51 865; a row that is read again when the bound
  // fails keeps its lines)
  template <bool STREAM> __device__ __forceinline__ void load() {
    if (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if ((int)threadIdx.x + i * NT < chunks) reg[i] = STREAM ? __builtin_nontemporal_load(body + threadIdx.x + i * NT) : body[threadIdx.x + i * NT];
    }
    if (extra_j >= 0) extra = (float)p[extra_j];
  }
  // element e of a chunk goes: an exponential of zero
  static __device__ __forceinline__ void without(V& v, int e) {
#pragma unroll
    for (int x = 0; x < N; ++x)
      if (x == e) v[x] = (E)-INFINITY;
  }
  // element j (e of chunk c, or -1: one of the ragged ends) goes from the registers: one wave has it
  __device__ __forceinline__ void drop(int j, int c, int e) {
    if (j >= 0 && extra_j == j) extra = -INFINITY;
    if (NC > 0 && c >= 0 && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) == c % NT >> 6) {
      const bool me = (int)threadIdx.x == c % NT;
      const uint32_t keep = N == 4 ? 0u : e & 1 ? 0xFFFFu : 0xFFFF0000u;
      const uint32_t put = N == 4 ? 0xFF800000u : (uint32_t)__builtin_bit_cast(uint16_t, (half_or<E>)-INFINITY) << (e & 1) * 16;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (i == c / NT) {
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (w == e * 4 / N) reg[i][w] = me ? (reg[i][w] & keep) | put : reg[i][w];
        }
    }
  }
  // f(chunk index, chunk).  The empty asm keeps hipcc from carrying the CONVERTED elements of one sweep over to the next (64 more registers per 8 chunks:
  // it spilled them).
  template <class F> __device__ __forceinline__ void each(F f) {
    if (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        if ((int)threadIdx.x + i * NT < chunks) {
          asm volatile("" : "+v"(reg[i]));
          f((int)threadIdx.x + i * NT, __builtin_bit_cast(V, reg[i]));
        }
      }
    } else {
      again(f);
    }
  }
  template <class F> __device__ __forceinline__ void again(F f) const {      // from memory
#pragma unroll 1
    for (int c = threadIdx.x; c < chunks; c += NT) f(c, __builtin_bit_cast(V, body[c]));
  }
};

// sum / maximum over NW neighbouring lanes, one per wave's entry
template <int NW, class T> __device__ __forceinline__ T over_waves(T v) {
#pragma unroll
  for (int o = NW / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int NW> __device__ __forceinline__ float max_over_waves(float v) {
#pragma unroll
  for (int o = NW / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float max_or_nan(float a, float b) { return b > a || b != b ? b : a; }
template <int NT> __device__ __forceinline__ float block_sum(float v, float* sh) {
  v = ns_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return over_waves<NT / 64>(sh[threadIdx.x & (NT / 64 - 1)]);
}
__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int NT> __device__ __forceinline__ int block_count(int v, int* sh) {
  v = wave_sum_int(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return over_waves<NT / 64>(sh[threadIdx.x & (NT / 64 - 1)]);
}
// a maximum to subtract: an infinite one is left in place of the difference (-inf: every exponential is zero; +inf: the sum becomes infinite)
__device__ __forceinline__ float finite_or_zero(float m) { return fabsf(m) == INFINITY ? 0.f : m; }

// ------------------------------------------------------------------------------------------------ the student
constexpr int DT_COUNT_HERE = 4;      // labels per thread that a row's workgroup counts itself (64 KB of L2 reads under its own row's loads) instead of a launch

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
  int rows, V, k, soft_only, count_here;
  float T, w1, w2, kd;
  float* row_loss; void* dz; int64_t lddz;
  int* nvalid; const float* loss_scale;
};

// DUAL: two softmaxes (0 < alpha < 1 at T != 1), else one, at T when only soft targets count.  2 and 4: the temperature is that, and e^z is a power of
// e^(z / T) by multiplication (its relative error T times the other's, which is what the argument's rounding in e^z itself amounts to).
// Per logit: a conversion and a maximum, then an fma, an exponential (a quarter-rate instruction) and an addition per softmax, and the same again for the
// gradient: with DUAL = 1 ~30 issue slots, 26 k cycles of a CU a row of 51 865 against the 20 k that the row's 208 KB take at the copy rate.
// A row that is almost certain of a token has 1 - p for a gradient there, which p itself does not hold: one token of the row, the label or the list's first entry, whichever has
// the larger logit, is left out of the sums, and 1 - p is what the others hold.
template <class E, int NC, int NT, int DUAL>
__global__ __launch_bounds__(NT, NT == 1024 && NC <= 7 ? 8 : 4) void distill_kernel(const DistillArgs p) {
  constexpr int NW = NT / 64;
  __shared__ float sh[3][NW];
  __shared__ int shc[NW];
  __shared__ __attribute__((aligned(16))) int sidx[DT_MAX_K + 4];
  __shared__ __attribute__((aligned(16))) float sp[DT_MAX_K + 4];
  __shared__ float sz[DT_MAX_K + 1];
  __shared__ float listed_rest;            // what the list gives to tokens other than the row's own
  typedef row_view<E, NC, NT> RV;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t lab64 = p.labels ? p.labels[row] : -1;
  const int listed = p.ti[row * p.ldt];      // (here, before any store, a scalar load: behind the row's loads it would wait for them, before them they for it)
  const bool has = lab64 >= 0 && lab64 < p.V;
  E* const out = p.dz ? (E*)p.dz + row * p.lddz : nullptr;
  RV r;
  r.init((const E*)p.z + row * p.ldz, p.V);
  const bool same = out && (((size_t)out ^ (size_t)r.p) & 15) == 0;
  ns_u4v* const obody = (ns_u4v*)(out + r.head);
  const bool dead = p.labels && !has;      // an ignored row: its logits are not read, its gradient is zero
  if (dead) {
    if (tid == 0) p.row_loss[row] = 0.f;
    if (out) {
      if (same) {
        for (int c = tid; c < r.chunks; c += NT) __builtin_nontemporal_store(ns_u4v{0, 0, 0, 0}, obody + c);
        if (r.extra_j >= 0) out[r.extra_j] = (E)0.f;
      } else {
        for (int j = tid; j < p.V; j += NT) out[j] = (E)0.f;
      }
    }
    if (!(p.count_here && row == 0)) return;
  }
  int live = 0;
  if (p.count_here)
    for (int i = tid; i < p.rows; i += NT) live += !p.labels || (p.labels[i] >= 0 && p.labels[i] < p.V);
  if (dead) {                              // (row 0 alone: it writes the count)
    live = wave_sum_int(live);
    if (lane == 0) shc[wave] = live;
    __syncthreads();
    if (tid == 0) {
      int n = 0;
      for (int w = 0; w < NW; ++w) n += shc[w];
      *p.nvalid = n;
    }
    return;
  }
  // the row's own token and its logit; it leaves the registers (its cell of the gradient is a sparse one).  (Both logits are asked for ahead of the row: behind it they cost a latency)
  const bool ok = listed >= 0 && listed < p.V;
  int own = has ? (int)lab64 : -1;
  const E z_label = r.p[has ? own : 0], z_listed = r.p[ok ? listed : 0];
  __builtin_amdgcn_sched_barrier(0);
  r.template load<true>();
  float zown = (float)z_label;
  {
    const float z = (float)z_listed;
    if (ok && !(has && zown >= z)) { own = listed; zown = z; }
    own = __builtin_amdgcn_readfirstlane(own);
    zown = __uint_as_float(__builtin_amdgcn_readfirstlane((int)__float_as_uint(zown)));
  }
  const int own_c = own >= r.head && own - r.head < r.chunks * RV::N ? (own - r.head) / RV::N : -1, own_e = (own - r.head) & (RV::N - 1);
  r.drop(own, own_c, own_e);
  // the lists: token, teacher logit / T, the student's logit there (read before any gradient overwrites it: dz may be z itself)
  for (int e = tid; e <= p.k; e += NT) {
    const int t = e == p.k ? (has ? (int)lab64 : -1) : p.ti[row * p.ldt + e];
    const bool ok = t >= 0 && t < p.V;
    sidx[e] = ok ? t : -1;
    sz[e] = ok ? (float)r.p[t] : 0.f;
    if (e < p.k) sp[e] = ok ? p.tv[row * p.ldt + e] / p.T : -INFINITY;
  }
  if (tid < 4) {                           // no entries behind the last (the sparse cells read four at a time)
    sp[p.k + tid] = 0.f;
    if (tid > 0) sidx[p.k + tid] = -1;
  }
  const float c1 = p.soft_only ? LOG2E / p.T : LOG2E, c2 = LOG2E / p.T;
  // every wave's maximum and sums relative to it, joined over the workgroup
  float mx = -INFINITY;
  r.each([&](int c, typename RV::V v) __attribute__((always_inline)) {
    if (NC == 0 && c == own_c) RV::without(v, own_e);
#pragma unroll
    for (int e = 0; e < RV::N; ++e) mx = fmaxf(mx, (float)v[e]);
  });
  mx = ns_wave_max(fmaxf(mx, r.extra));
  float s1 = 0.f, s2 = 0.f;
  {
    const float m = finite_or_zero(mx);      // (subtracted first: a maximum near the type's lowest value times c would overflow)
    auto add = [&](float x) __attribute__((always_inline)) {
      if (DUAL < 2) s1 += __builtin_amdgcn_exp2f((x - m) * c1);
      if (DUAL) {
        const float y = __builtin_amdgcn_exp2f((x - m) * c2), y2 = y * y;
        s2 += y;
        if (DUAL == 2) s1 += y2;
        if (DUAL == 4) s1 = __builtin_fmaf(y2, y2, s1);
      }
    };
    r.each([&](int c, typename RV::V v) __attribute__((always_inline)) {
      if (NC == 0 && c == own_c) RV::without(v, own_e);
#pragma unroll
      for (int e = 0; e < RV::N; ++e) add((float)v[e]);
    });
    add(r.extra);
  }
  s1 = ns_wave_sum(s1);
  if (DUAL) s2 = ns_wave_sum(s2);
  if (p.count_here) live = wave_sum_int(live);
  if (lane == 0) { sh[0][wave] = mx; sh[1][wave] = s1; sh[2][wave] = s2; shc[wave] = live; }
  __syncthreads();                         // also: sz[] has been read from z by everyone who reads it
  const int ent = lane & (NW - 1);
  const float wm = sh[0][ent];
  mx = max_over_waves<NW>(wm);
  if (own >= 0) mx = fmaxf(mx, zown);
  const float ms = finite_or_zero(mx), dm = wm == -INFINITY ? -INFINITY : finite_or_zero(wm) - ms;      // (a wave without elements, or of -inf: no part)
  s1 = over_waves<NW>(sh[1][ent] * __builtin_amdgcn_exp2f(dm * c1));
  if (DUAL) s2 = over_waves<NW>(sh[2][ent] * __builtin_amdgcn_exp2f(dm * c2));
  // x1, x2: a logit's part of the two sums
  auto parts = [&](float z, float& x1, float& x2) __attribute__((always_inline)) {
    x2 = DUAL ? __builtin_amdgcn_exp2f((z - ms) * c2) : 0.f;
    x1 = DUAL == 2 ? x2 * x2 : DUAL == 4 ? (x2 * x2) * (x2 * x2) : __builtin_amdgcn_exp2f((z - ms) * c1);
  };
  float rest1 = 1.f, rest2 = 1.f;          // 1 - p, 1 - q of the row's own token
  if (own >= 0) {
    float x1, x2;
    parts(zown, x1, x2);
    rest1 = __builtin_fmaf(0.f, x1, s1 / (s1 + x1));      // (an infinity shows)
    s1 += x1;
    rest2 = DUAL ? __builtin_fmaf(0.f, x2, s2 / (s2 + x2)) : rest1;
    s2 += x2;
  }
  live = over_waves<NW>(shc[ent]);
  if (p.count_here) { if (row == 0 && tid == 0) *p.nvalid = live; }
  else live = *p.nvalid;
  // the teacher's distribution: every wave forms its maximum, the first one the row's loss and the probabilities
  float tm = -INFINITY;
  for (int e = lane; e < p.k; e += 64) tm = max_or_nan(tm, sp[e]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) tm = max_or_nan(tm, __shfl_xor(tm, o, 64));
  const bool soft = tm != -INFINITY;       // a list that names no token leaves the hard label alone; a NaN or +inf that an entry holds shows in the row's loss
  __syncthreads();                         // every wave has read sp[] before the first one turns it into probabilities
  if (wave == 0) {
    float ts = 0.f;
    for (int e = lane; e < p.k; e += 64) ts += soft ? expf(sp[e] - tm) : 0.f;
    ts = ns_wave_sum(ts);
    const float lt = logf(ts), its = 1.f / ts, ls = logf(DUAL ? s2 : s1);
    float kl = 0.f, lr = 0.f;
    for (int e = lane; e < p.k; e += 64) {
      const float lp = sp[e] - tm;
      const float pr = soft ? expf(lp) * its : 0.f;
      if (pr != 0.f) kl += pr * ((lp - lt) - ((sz[e] - ms) / p.T - ls));
      sp[e] = pr;
      lr += sidx[e] == own ? 0.f : pr;
    }
    kl = ns_wave_sum(kl);
    lr = ns_wave_sum(lr);
    if (lane == 0) {
      listed_rest = lr;
      float loss = soft ? p.kd * kl : 0.f;
      if (!p.soft_only) loss += p.w1 * ((ms - sz[p.k]) + logf(s1));
      p.row_loss[row] = loss;
    }
  }
  if (!out) return;
  // the gradient's weights ride in the exponents: g w 2^((z - m) c) / s = 2^((z - m) c - (log2 s - log2(g w))); a weight of zero is an exponent of -inf
  const float gs = (p.loss_scale ? *p.loss_scale : 1.f) / (float)max(live, 1);
  const float w2 = soft ? p.w2 : 0.f;
  const float f1 = fabsf(gs) * (DUAL ? p.w1 : (p.soft_only ? 0.f : p.w1) + w2), f2 = fabsf(gs) * w2;
  const float a1 = log2f(s1) - log2f(f1), a2 = DUAL ? log2f(s2) - log2f(f2) : 0.f;
  const float sign = gs < 0.f ? -1.f : 1.f;
  const float k1 = gs * p.w1 / s1, k2 = gs * w2 / s2;      // (DUAL 2, 4)
  auto grad = [&](float z) __attribute__((always_inline)) {
    const float x = z - ms;
    if (DUAL >= 2) {
      const float y = __builtin_amdgcn_exp2f(x * c2);
      return y * __builtin_fmaf(DUAL == 2 ? y : y * y * y, k1, k2);
    }
    float g = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c1, -a1));
    if (DUAL) g += __builtin_amdgcn_exp2f(__builtin_fmaf(x, c2, -a2));
    return g * sign;
  };
  if (same) {
    r.each([&](int c, typename RV::V v) __attribute__((always_inline)) {
      typename RV::V o;
#pragma unroll
      for (int e = 0; e < RV::N; ++e) o[e] = (E)grad((float)v[e]);
      __builtin_nontemporal_store(__builtin_bit_cast(ns_u4v, o), obody + c);
    });
  } else {
    r.again([&](int c, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < RV::N; ++e) out[r.head + c * RV::N + e] = (E)grad((float)v[e]);
    });
  }
  if (r.extra_j >= 0) out[r.extra_j] = (E)grad(r.extra);
  // the sparse cells, each token once whatever number of entries name it, behind the dense stores
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (int e = tid; e <= p.k; e += NT) {
    const int t = sidx[e];
    if (t < 0) continue;
    float q = 0.f;
    bool first = true;
#pragma unroll 4
    for (int o = 0; o < p.k; o += 4) {     // (sp[k] is zero, and entry k comes no earlier than any)
      const int4 s = *(const int4*)&sidx[o];
      const float4 r4 = *(const float4*)&sp[o];
      q += (s.x == t ? r4.x : 0.f) + (s.y == t ? r4.y : 0.f) + (s.z == t ? r4.z : 0.f) + (s.w == t ? r4.w : 0.f);
      first = first && !((s.x == t && o < e) || (s.y == t && o + 1 < e) || (s.z == t && o + 2 < e) || (s.w == t && o + 3 < e));
    }
    if (!first) continue;
    const bool label = has && t == (int)lab64;
    float x1, x2;
    parts(sz[e], x1, x2);
    // where the row is certain of this token: p - 1 = -(1 - p), q - t = (1 - t) - (1 - q)
    const float d1 = t == own && rest1 < 0.5f ? (label ? -rest1 : 1.f - rest1) : x1 / s1 - (label ? 1.f : 0.f);
    const float d2 = t == own && rest2 < 0.5f ? listed_rest - rest2 : (DUAL ? x2 / s2 : x1 / s1) - q;
    out[t] = (E)(gs * ((p.soft_only ? 0.f : p.w1 * d1) + (soft ? w2 * d2 : 0.f)));
  }
}

// ------------------------------------------------------------------------------------------------ the teacher
// The k largest of a row.  Every thread's largest element is put into one of BINS equal bins between the smallest and the largest of those; the bin
// that the k-th largest of them falls into is a bound that at least k elements reach and few more: the elements in that bin or above it are collected
// (only in chunks whose own maximum reaches it) and ordered by (value, lowest token first).  If more than CAP reach it -- rows of equal values -- or
// the row holds an infinity or a NaN, the k-th largest value is found bit by bit over all elements, then the token below which enough elements EQUAL to it
// lie: exactly k remain (up to 64 sweeps of the row).  A NaN ranks above +inf.
// 4096 fp16 rows of 51 865, k = 64: 117 - 126 us; bit by bit 4.5 ms where all values are equal, 0.6 ms where one value lies so far above the rest that they share a bin (far below, or
// -inf in half of the tokens: 117).  A short row of which fewer than k threads hold elements and more than CAP elements are offered goes that way too: 1500 tokens, k = 64: 20 us, k = 200: 204.
__device__ __forceinline__ uint32_t order_key(float x) {
  const float f = x + 0.f;                             // -0 ranks as +0
  const uint32_t u = __float_as_uint(f);
  if (f != f) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <class E, int NC, int NT>
__global__ __launch_bounds__(NT, NT == 1024 && NC <= 7 ? 8 : 4) void topk_row_kernel(const E* __restrict__ z, int64_t ldz, int V, int k,
                                                                                              float* __restrict__ vals, int32_t* __restrict__ idx,
                                                                                              int64_t ldo, float* __restrict__ lse) {
  constexpr int CAP = 1024, BINS = 256, NW = NT / 64;
  __shared__ uint64_t cand[CAP];
  __shared__ int hist[BINS];
  __shared__ int shi[NW];
  __shared__ float sh[3][NW];
  __shared__ int count, bound_bin;
  typedef row_view<E, NC, NT> RV;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  RV r;
  r.init(z + row * ldz, V);
  r.template load<false>();
  for (int b = tid; b < BINS; b += NT) hist[b] = 0;
  if (tid == 0) count = 0;
  const bool some = tid < r.chunks || r.extra_j >= 0;         // this thread holds elements
  float mx = -INFINITY;
  r.each([&](int, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < RV::N; ++e) mx = fmaxf(mx, (float)v[e]);
  });
  mx = fmaxf(mx, r.extra);
  const float wmx = ns_wave_max(mx);
  const float wmn = -ns_wave_max(some ? -mx : -INFINITY);
  float s = 0.f;
  {
    const float m = finite_or_zero(wmx);
    r.each([&](int, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < RV::N; ++e) s += __builtin_amdgcn_exp2f(((float)v[e] - m) * LOG2E);
    });
    s += __builtin_amdgcn_exp2f((r.extra - m) * LOG2E);
    s = ns_wave_sum(s);
  }
  if (lane == 0) { sh[0][wave] = wmx; sh[1][wave] = wmn; sh[2][wave] = s; }
  __syncthreads();
  const int ent = lane & (NW - 1);
  const float wm = sh[0][ent];
  const float hi = max_over_waves<NW>(wm), lo = -max_over_waves<NW>(-sh[1][ent]);
  const float ms = finite_or_zero(hi);
  s = over_waves<NW>(sh[2][ent] * (wm == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((finite_or_zero(wm) - ms) * LOG2E)));
  if (lse && tid == 0) lse[row] = ms + logf(s);
  // a bin is a monotone function of the value: rounding keeps the order.  (hi == lo: one bin.)
  const bool plain = s == s && fabsf(hi) < INFINITY && fabsf(lo) < INFINITY;
  const float scale = hi > lo ? (float)(BINS - 1) / (hi - lo) : 0.f;
  auto bin = [&](float x) __attribute__((always_inline)) { return x >= lo ? min((int)((x - lo) * scale), BINS - 1) : -1; };
  int n = CAP + 1;
  if (plain && scale < INFINITY) {
    if (some) atomicAdd(&hist[bin(mx)], 1);
    __syncthreads();
    if (wave == 0) {                                          // the highest bin that, with those above it, holds k thread maxima (-1: fewer than k threads)
      int own[4], sum = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) { own[b] = hist[lane * 4 + b]; sum += own[b]; }
      int above = 0;                                          // in the bins of higher lanes
      int run = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_down(run, o, 64);
        run += lane + o < 64 ? t : 0;
      }
      above = run - sum;
      int at = -1;
#pragma unroll
      for (int b = 3; b >= 0; --b) {
        above += own[b];
        if (at < 0 && above >= k) at = lane * 4 + b;
      }
      at = (int)ns_wave_max((float)at);
      if (lane == 0) bound_bin = at;
    }
    __syncthreads();
    const int bb = bound_bin;
    auto offer = [&](float x, int at) __attribute__((always_inline)) {
      if (bin(x) < bb) return;
      const int to = atomicAdd(&count, 1);
      if (to < CAP) cand[to] = ((uint64_t)order_key(x) << 32) | (uint32_t)~at;
    };
    r.each([&](int c, typename RV::V v) __attribute__((always_inline)) {
      float cm = (float)v[0];
#pragma unroll
      for (int e = 1; e < RV::N; ++e) cm = fmaxf(cm, (float)v[e]);
      if (bin(cm) >= bb) {
#pragma unroll
        for (int e = 0; e < RV::N; ++e) offer((float)v[e], r.head + c * RV::N + e);
      }
    });
    if (r.extra_j >= 0) offer(r.extra, r.extra_j);
    __syncthreads();
    n = count;
  }
  if (n > CAP) {
    auto reach = [&](auto take) __attribute__((always_inline)) {
      int c = r.extra_j >= 0 && take(order_key(r.extra), r.extra_j) ? 1 : 0;
      r.again([&](int at, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < RV::N; ++e) c += take(order_key((float)v[e]), r.head + at * RV::N + e);
      });
      return block_count<NT>(c, shi);
    };
    uint32_t kth = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = kth | (1u << b);
      if (reach([&](uint32_t key, int) { return key >= t; }) >= k) kth = t;
    }
    const int more = reach([&](uint32_t key, int) { return key > kth; });
    int upto = 0;                                             // the largest bound below which fewer than k - more equal elements lie
#pragma unroll 1
    for (int b = 30; b >= 0; --b) {
      const int t = upto | (1 << b);
      if (reach([&](uint32_t key, int at) { return key == kth && at < t; }) < k - more) upto = t;
    }
    __syncthreads();
    if (tid == 0) count = 0;
    __syncthreads();
    auto keep = [&](float x, int at) __attribute__((always_inline)) {
      const uint32_t key = order_key(x);
      if (key > kth || (key == kth && at <= upto)) cand[atomicAdd(&count, 1)] = ((uint64_t)key << 32) | (uint32_t)~at;
    };
    r.again([&](int c, typename RV::V v) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < RV::N; ++e) keep((float)v[e], r.head + c * RV::N + e);
    });
    if (r.extra_j >= 0) keep(r.extra, r.extra_j);
    __syncthreads();
    n = count;                                                // exactly k
  }
  // each candidate's place is the number of candidates above it: eight lanes a candidate
  const int sub = tid & 7;
  for (int c = tid >> 3; c < n; c += NT / 8) {
    const uint64_t me = cand[c];
    int above = 0;
    for (int o = sub; o < n; o += 8) above += cand[o] > me;
    above += __shfl_xor(above, 1, 64);
    above += __shfl_xor(above, 2, 64);
    above += __shfl_xor(above, 4, 64);
    if (sub == 0 && above < k) {
      const int t = (int)~(uint32_t)me;
      vals[row * ldo + above] = (float)r.p[t];
      idx[row * ldo + above] = t;
    }
  }
}

template <class E, template <class, int, int> class Launch, class... A>
void by_length(int V, A... a) {
  // threads and registers by the row's length: one or two accesses a thread on 256 threads, then 1024 threads with as many as the row needs; up to seven
  // (28 registers) two workgroups share a CU, so that one loads while the other computes
  const int chunks = V / vec<E>::N;
  if (chunks <= 256) Launch<E, 1, 256>::go(a...);
  else if (chunks <= 512) Launch<E, 2, 256>::go(a...);
  else if (chunks <= 2 * 1024) Launch<E, 2, 1024>::go(a...);
  else if (chunks <= 4 * 1024) Launch<E, 4, 1024>::go(a...);
  else if (chunks <= 7 * 1024) Launch<E, 7, 1024>::go(a...);
  else if (sizeof(E) == 4 && chunks <= 14 * 1024) Launch<E, sizeof(E) == 4 ? 14 : 0, 1024>::go(a...);
  else Launch<E, 0, 1024>::go(a...);
}

template <class E, int NC, int NT> struct distill_go {
  static void go(DistillArgs a, bool dual, hipStream_t st) {
    a.count_here = a.rows <= DT_COUNT_HERE * NT;
    if (!a.count_here) hipLaunchKernelGGL(dt_count_kernel, dim3(1), dim3(1024), 0, st, a.labels, a.rows, a.V, a.nvalid);
    if (!dual) hipLaunchKernelGGL((distill_kernel<E, NC, NT, 0>), dim3(a.rows), dim3(NT), 0, st, a);
    else if (a.T == 2.f) hipLaunchKernelGGL((distill_kernel<E, NC, NT, 2>), dim3(a.rows), dim3(NT), 0, st, a);
    else if (a.T == 4.f) hipLaunchKernelGGL((distill_kernel<E, NC, NT, 4>), dim3(a.rows), dim3(NT), 0, st, a);
    else hipLaunchKernelGGL((distill_kernel<E, NC, NT, 1>), dim3(a.rows), dim3(NT), 0, st, a);
  }
};
template <class E, int NC, int NT> struct topk_go {
  static void go(const ns_topk_desc* d, hipStream_t st) {
    hipLaunchKernelGGL((topk_row_kernel<E, NC, NT>), dim3(d->rows), dim3(NT), 0, st, (const E*)d->logits, d->ldz, d->vocab, d->k, d->vals, d->idx, d->ldo, d->lse);
  }
};

// a launch holds less than 2^32 threads: by_length's workgroups, one a row
bool rows_fit(int rows, int V, int dtype) { return (int64_t)rows * ((V / (dtype == NS_F32 ? 4 : 8) <= 512) ? 256 : 1024) < (1ll << 32); }

bool elem_aligned(const void* q, int dtype) { return ((size_t)q & (dtype == NS_F32 ? 3 : 1)) == 0; }

}  // namespace

extern "C" int ns_distill_topk(const ns_distill_desc* d, void* stream) {
  NS_CHECK_ARG(d, "ns_distill_topk: null descriptor");
  NS_CHECK_ARG(d->loss_dev && d->nvalid_dev && (d->rows == 0 || (d->logits && d->row_loss && d->top_vals && d->top_idx)), "ns_distill_topk: null pointer");
  NS_CHECK_ARG(d->rows >= 0 && d->vocab > 0 && d->vocab <= (1 << 30) && d->k > 0 && d->k <= DT_MAX_K, "ns_distill_topk: bad sizes rows=%d vocab=%d k=%d (k <= %d)", d->rows,
               d->vocab, d->k, DT_MAX_K);
  NS_CHECK_ARG(d->dtype == NS_F16 || d->dtype == NS_BF16 || d->dtype == NS_F32, "ns_distill_topk: dtype %d", d->dtype);
  NS_CHECK_ARG(rows_fit(d->rows, d->vocab, d->dtype), "ns_distill_topk: rows=%d are too many for one launch", d->rows);
  NS_CHECK_ARG(d->rows <= 1 || (d->ldz >= d->vocab && d->ld_top >= d->k && (!d->dlogits || d->lddz >= d->vocab)), "ns_distill_topk: row strides shorter than the rows");
  NS_CHECK_ARG(elem_aligned(d->logits, d->dtype) && elem_aligned(d->dlogits, d->dtype), "ns_distill_topk: logits not aligned to their elements");
  NS_CHECK_ARG(d->temperature >= 0.05f && d->temperature <= 100.f && d->alpha > 0.f && d->alpha <= 1.f, "ns_distill_topk: temperature %g in [0.05, 100], alpha %g in (0, 1]",
               (double)d->temperature, (double)d->alpha);
  NS_CHECK_ARG(d->labels || d->alpha == 1.f || d->rows == 0, "ns_distill_topk: alpha %g < 1 needs labels", (double)d->alpha);
  hipStream_t st = (hipStream_t)stream;
  if (d->rows > 0) {
    DistillArgs a = {};
    a.z = d->logits; a.ldz = d->ldz; a.labels = d->labels; a.tv = d->top_vals; a.ti = d->top_idx; a.ldt = d->ld_top; a.rows = d->rows; a.V = d->vocab; a.k = d->k;
    a.soft_only = d->alpha == 1.f;
    const bool dual = !a.soft_only && d->temperature != 1.f;
    a.T = d->temperature; a.w1 = 1.f - d->alpha; a.w2 = d->alpha * d->temperature; a.kd = d->alpha * d->temperature * d->temperature;
    a.row_loss = d->row_loss; a.dz = d->dlogits; a.lddz = d->lddz; a.nvalid = d->nvalid_dev; a.loss_scale = d->loss_scale_dev;
    if (d->dtype == NS_F16) by_length<half_t, distill_go>(d->vocab, a, dual, st);
    else if (d->dtype == NS_BF16) by_length<__bf16, distill_go>(d->vocab, a, dual, st);
    else by_length<float, distill_go>(d->vocab, a, dual, st);
  } else {
    hipLaunchKernelGGL(dt_count_kernel, dim3(1), dim3(1024), 0, st, d->labels, 0, d->vocab, d->nvalid_dev);
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
  NS_CHECK_ARG(rows_fit(d->rows, d->vocab, d->dtype), "ns_topk_logits: rows=%d are too many for one launch", d->rows);
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
