// ns_linear_cross_entropy: the LM head and its loss in one call, without the (rows, vocabulary) logits.
//
//   z = h W^T                                       h (N, d) hidden states, W (V, d) the head
//   CE_i = lse(z_i) - z_i[label_i]
//   KL_i = sum_k p_ik (log p_ik - (z_i[idx_ik] / T - lse(z_i / T))),      p_i = softmax of the teacher's top logits / T
//   loss = mean over the rows with a label of (1 - alpha) CE_i + alpha T^2 KL_i
//   dz_i = g [ w1 softmax(z_i) + w2 softmax(z_i / T) - w1 onehot(label_i) - w2 sum_k p_ik onehot(idx_ik) ],   w1 = 1 - alpha, w2 = alpha T
//   dh = dz W,  dW = dz^T h,                        g = loss_scale / rows with a label
//
// The logits pass through the registers of 256 x 256 MFMA tiles and are never stored as such.  One pass keeps the running maximum and sum of every row (fp32,
// one pair per row and 256 columns, joined by ll_rows_kernel).  dz in the operands' type then lies in a workspace, from where the products dh = dz W and
// dW = dz^T h take it.  It comes about in one of two ways:
//   kept     the same pass leaves 2^(z - reference): no logit is formed twice.  With one reference for the row, taken from its label's logit, this is dz but for the
//            row's factor (one softmax; bf16, or dh alone from labels: see ll_label_ref); else the reference is that of the row's 64-column strip and ll_scale_kernel
//            makes dz of it in place.  One softmax (or two at 1 <= T <= 2), and whole rows.  Where dW is not asked for, chunks of rows one after the other, each within LL_PIECE_BYTES (it stays in the
//            256-MiB last-level cache); dW needs all rows, at most LL_WHOLE_BYTES of them.
//   formed again   a second pass over the logits writes dz of one PIECE of the vocabulary (LL_PIECE_BYTES) for all rows, piece after piece: 4 products instead of 3,
//            but no more memory, and dW, of V d elements, is written once (chunks of rows would read and write it per chunk).
//            8192 rows, d = 1280, V = 51865, bf16, dh and dW: 3.59 ms formed again in 256 MiB, 2.72 ms kept in 852 MB; 1434 rows, d = 512, fp16, a list: 432 us at T = 4, 397 at T = 1.5.
//   * Rows without a label are packed away first: they cost nothing, and an infinity or NaN in a masked row reaches neither loss nor gradient.
//   * A row's sparse terms (its label, the teacher's list) are no part of the dense epilogue: their logits are gathered as dot products in fp32
//     and their cells of dz are written from those.  One of them a row, its own token, is no part of the statistics either: 1 - p of a row that is almost certain is
//     then a sum of its own, not what is left of p (ll_rows_kernel).
//   * dz in the operands' type: fp16 cells carry a factor 2^s (exact; taken out in fp32 at the end), so that a probability of 1 / V does
//     not fall among the subnormals; a probability below 2^-29 of full scale is a subnormal, below 2^-40 zero (dh alone from labels: of what the other tokens hold, see
//     ll_label_ref).  bf16 has the range of fp32.
//     A sparse cell is rounded once, after the subtraction, a kept one twice (its exponential, dz).  A row's largest cells count by themselves: with up to 32 labels
//     a cell is two numbers, up to 64 what the largest cell in each 256 tokens lost is added in fp32 (ll_few_grad), beyond 64 rows dh's and dW's last steps add what the two
//     largest lost (ll_cells_kernel) or all of them (ll_label_ref).
//   * Sums over the vocabulary (dh) and over the rows (dW) stay in fp32 MFMA accumulators / fp32 tiles added in a fixed order: no atomics
//     (but a maximum in LDS), the same bits every time.
//   * What bounds it: the 256 x 256 main loops (8 waves, two 64 KiB ring buffers, one workgroup per CU) take 2.9 k cycles per K tile of 64 against 2.05 k of MFMA: a K tile's
//     fragments and DMA are 256 KiB, another 2 k cycles of the LDS port, and the two overlap in part.  At d = 1280 a launch reaches 1.1 (logits, with the exponentials) to
//     1.3 PFLOP/s (dh, dW), the matrix pipes 0.54 - 0.68 busy at a clock that falls to 1.8 - 2.0 GHz (a plain library product of the shape: 1.1 - 1.3); at d = 512, with eight
//     K tiles to an epilogue, 0.7 - 0.9, the pipes 0.36 - 0.52 busy at 2.25 GHz.
// The 256 x 256 main loop is ns_gemm_p8.hip's four-phase LDS-DMA ring (see there: two wave groups one barrier interval apart), here for both
// 16-bit types and with a second operand that may be K-major (W for dh, dz for dW): such a region holds 64 k-rows of 256 B and its fragments are
// read transposed by ds_read_b64_tr_b16.
#include "ns_common.h"

namespace {

constexpr int BM = 256, BN = 256, BK = 64, NTH = 512;
constexpr int REGION = 128 * 128;            // 16 KiB
constexpr int BUF = 4 * REGION;              // 64 KiB
constexpr int RA0 = 0, RA1 = 1, RB0 = 2, RB1 = 3;
constexpr int LDH = BN * 2 + 16;             // epilogue: bytes per staged 16-bit row
constexpr int LL_LDS = BM * LDH > 2 * BUF ? BM * LDH : 2 * BUF;      // (also what every kernel's attribute allows)
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr size_t LL_PIECE_BYTES = 256u << 20, LL_WHOLE_BYTES = 1u << 30;
constexpr int LL_MAX_K = 256;
constexpr uint32_t OUT = 0x80000000u;        // a buffer offset past every resource: the hardware returns zeros

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef unsigned short ushort4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v lds_s4;

struct tf16 {
  static constexpr float HEAD = 15.f, BELOW = 6.f, LOW = -14.f;       // (see ll_label_ref)
  typedef half_t e;
  typedef half8 v8;
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
struct tbf16 {
  static constexpr float HEAD = 30.f, BELOW = 0.f, LOW = -INFINITY;
  typedef __bf16 e;
  typedef bf8 v8;
  static __device__ __forceinline__ f32x4 mma(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <class E> __device__ __forceinline__ ushort4v cvt4(float a, float b, float c, float d) {
  typedef E e4 __attribute__((ext_vector_type(4)));
  const e4 r = {(E)a, (E)b, (E)c, (E)d};
  return __builtin_bit_cast(ushort4v, r);
}

// A DMA piece in asm: behind the builtin hipcc waits for every piece in flight (vmcnt(0)) before a transposed LDS read, which it takes to alias
// them; the ring's own counted waits order the two.  The instruction has no register result.
__device__ __forceinline__ void ll_dma16(ns_u4v rsrc, uint32_t voff, int soff, uint32_t lds_dst) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(voff), "s"(rsrc), "s"(soff), "s"(lds_dst) : "memory");
}
__device__ __forceinline__ ns_u4v ll_rsrc(const void* base) {
  const uint64_t a = (uint64_t)base;
  return ns_u4v{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)), OUT, 0x00020000u};
}

// reductions over the four lanes that are 16 apart (equal lane & 15): the swap instructions exchange 16-lane rows / 32-lane halves of two copies
__device__ __forceinline__ void ll_swap(float v, bool by32, float& a, float& b) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 r = by32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false)
                    : __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  a = __uint_as_float(r[0]);
  b = __uint_as_float(r[1]);
}
__device__ __forceinline__ float ll_max4(float v) {
  float a, b;
  ll_swap(v, false, a, b);
  v = fmaxf(a, b);
  ll_swap(v, true, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float ll_sum4(float v) {
  float a, b;
  ll_swap(v, false, a, b);
  v = a + b;
  ll_swap(v, true, a, b);
  return a + b;
}

// reference exponent of a softmax at scale c: an integer, so that taking it out of z c (inside the fma) and moving sums between references are exact
__device__ __forceinline__ float ll_ref(float mx, float c) { return ceilf(mx * c); }

// LL_KEEP with one reference for a whole row (REF: one softmax).  The label's logit is known before the pass: its exponent (less BELOW, which moves fp16's range)
// is the row's reference as long as no logit but the label's exceeds it by more than 2^HEAD.  A 64-column strip that does exceed it takes its own maximum, and its row is brought to
// one reference afterwards.  So dz = x F with ONE factor per row, which dh's last step and h's transposed copy take in, and the pass over dz falls away
// (bf16, 8192 rows, d = 1280: 2.93 -> 2.72 ms; 1844 rows, d = 512: 425 -> 382 us; fp16, 1229 rows, dh alone: 218 -> 173 us, and 204 where
// every row's reference changes, as with labels that are almost certain).
//   bfloat16   has the exponents for x and for the cells of a list, up to 2^47; what lies 2^-126 below the label counts for nothing.
//   float16    has room for x alone, up to 2^9 times the label's, and none for h's copy with the factors: dh alone, and no list.  Below 2^LOW its numbers lose digits, by at
//              most 2^-25 each: where the label is almost certain, all that is left of the row's gradient lies there.  So a strip is kept relative to the label only if its
//              largest x is at least 64 2^LOW, else to its own maximum (either way the strip as a whole is within 2^-11 of itself), and a row of which the V others do not hold
//              V 2^LOW together goes to the reference of their largest, as one whose largest exceeds 2^HEAD does (2^-39 V of what they hold, at most, is lost there).
// Without a list the label's x is zero (it is the row's own token), and dh's and dW's last steps add (p - 1) W[label] and (p - 1) h in fp32: a rounded factor or cell would be an error of all of
// a row's gradient, and subtracting W[label] from a product that holds p W[label] would leave p's rounding of 1 - p.
// The gathered logit and the tile's differ by the order of their sums, each within (d + 4) u sum |h w| of the exact one: where that could exceed 4 the row gets no
// reference (NaN: every comparison fails).
template <class T> __device__ __forceinline__ float ll_label_ref(float z, float mass, int d, float c) {
  return (float)(d + 4) * 5.9604645e-8f * mass * c <= 4.f ? ll_ref(z, c) - T::BELOW : NAN;
}
template <class T> __device__ __forceinline__ float ll_strip_ref(float mx, float eref, float c, float shift) {
  return mx * c <= eref + T::HEAD && mx * c >= eref + T::LOW + 6.f ? eref : mx == -INFINITY ? 0.f : ll_ref(mx, c) - shift;
}

#define LL_BARRIER()                            \
  do {                                          \
    asm volatile("" ::: "memory");              \
    __builtin_amdgcn_s_barrier();               \
    asm volatile("" ::: "memory");              \
  } while (0)

// One 256 x 256 tile, C = A B over `K`: A rows are K-contiguous; B is K-contiguous (BT = false: rows n) or K-major (BT = true: rows k).
// a_base / b_base: first element of the tile's operand (row m0 / row n0, or column n0 of k-row 0); ld in elements, extents from there < 2 GiB.
// kA / kB: valid k of each operand (chunks / k-rows past them are zeros); b_rows: valid rows n (BT = false) or columns n (BT = true), a multiple of 8 when BT.
// SWAP = false: a lane owns 4 consecutive n of row m = l15 (acc[..][reg]); SWAP = true: 4 consecutive m of column n = l15.
template <class T, bool BT, bool SWAP>
__device__ __forceinline__ void ll_tile(f32x4 (&acc)[2][4][2][2], char* smem, const void* a_base, int lda, int kA,
                                        const void* b_base, int ldb, int kB, int b_rows, int K) {
  typedef typename T::v8 v8;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int l15 = lane & 15, lg = lane >> 4;
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[a][i][b][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // DMA sources: wave w fills region bytes [2048 w, 2048 w + 2048) as two 1-KiB pieces.  K-contiguous: 8 rows x 128 B, chunk c of region row r
  // holds source chunk c ^ ((r >> 1) & 7).  K-major: 4 k-rows x 256 B, the 32-B windows of k-row r are permuted by g(r) = (r & 3) | ((r >> 3) & 1) << 2:
  // the eight row segments that half a wave reads transposed (four k-rows of two 16-lane groups, 8 k-rows apart) lie in eight different windows.
  uint32_t a_off[2][2], b_off[2][2];
  int a_k[2], b_k[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int rr = 16 * wave + 8 * j + (lane >> 3);
    const int ch = (lane & 7) ^ ((rr >> 1) & 7);
    a_k[j] = ch * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int arow = ((rr >> 6) << 7) + h * 64 + (rr & 63);
      a_off[h][j] = (uint32_t)(arow * lda + ch * 8) * 2u;
      if (!BT) {
        const int brow = ((rr >> 5) << 6) + h * 32 + (rr & 31);
        b_off[h][j] = brow < b_rows ? (uint32_t)(brow * ldb + ch * 8) * 2u : OUT;
      }
    }
    b_k[j] = ch * 8;
    if (BT) {
      const int kr = 8 * wave + 4 * j + (lane >> 4);
      const int g = (kr & 3) | (((kr >> 3) & 1) << 2);
      const int col = ((lane & 15) ^ (g << 1)) * 8;        // region column 0 .. 127
      b_k[j] = kr;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = ((col >> 5) << 6) + h * 32 + (col & 31);
        b_off[h][j] = n < b_rows ? (uint32_t)(kr * ldb + n) * 2u : OUT;
      }
    }
  }
  const ns_u4v rsrc_a = ll_rsrc(a_base), rsrc_b = ll_rsrc(b_base);
  const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)smem;
  auto stage = [&](int tt, int region, int buf) __attribute__((always_inline)) {
    const int k0 = tt * BK, h = region & 1;
    const bool isb = region >= 2;
    const int klen = (isb ? kB : kA) - k0;
    const int soff = isb ? (BT ? k0 * ldb * 2 : k0 * 2) : k0 * 2;
    const uint32_t dst = lds_base + buf * BUF + region * REGION + wave * 2048;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool ok = (isb ? b_k[j] : a_k[j]) < klen;
      const uint32_t off = isb ? b_off[h][j] : a_off[h][j];
      // (a tile past the end asks for nothing: offset and scalar offset must not wrap around together)
      ll_dma16(isb ? rsrc_b : rsrc_a, ok ? off : OUT, klen > 0 ? soff : 0, dst + j * 1024);
    }
  };
  const int fsw = ((lg ^ (l15 >> 1)) & 7) << 4;
  const int a_rd = (wm * 64 + l15) * 128 + fsw;
  const int q = l15 >> 2, pp = l15 & 3;
  const int b_rd = BT ? (8 * lg + q) * 256 + (((wn * 2) ^ (q | ((lg & 1) << 2))) << 5) + pp * 8 : (wn * 32 + l15) * 128 + fsw;

  v8 af[4][2], bq[2][2][2];
  auto read_a = [&](int buf, int ah) __attribute__((always_inline)) {
    const char* st = smem + buf * BUF + (ah ? RA1 : RA0) * REGION;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) af[mt][ks] = *(const v8*)(st + ((a_rd ^ (ks << 6)) + mt * 2048));
  };
  auto read_b = [&](int buf, int bh) __attribute__((always_inline)) {
    const char* st = smem + buf * BUF + (bh ? RB1 : RB0) * REGION;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (!BT) {
          bq[bh][nt][ks] = *(const v8*)(st + ((b_rd ^ (ks << 6)) + nt * 2048));
        } else {
          const char* const at = st + ((b_rd ^ (nt << 5)) + ks * 8192);
          const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
          const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 1024));
          const short8v r = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          bq[bh][nt][ks] = __builtin_bit_cast(v8, r);
        }
      }
  };
  auto mma = [&](int ah, int bh) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
          acc[ah][mt][bh][nt] = SWAP ? T::mma(af[mt][ks], bq[bh][nt][ks], acc[ah][mt][bh][nt]) : T::mma(bq[bh][nt][ks], af[mt][ks], acc[ah][mt][bh][nt]);
    __builtin_amdgcn_s_setprio(0);
  };
#define LL_RUN(AH, BH)                                      \
  do {                                                      \
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");        \
    LL_BARRIER();                                           \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      \
    __builtin_amdgcn_sched_barrier(0);                      \
    mma(AH, BH);                                            \
    __builtin_amdgcn_sched_barrier(0);                      \
    LL_BARRIER();                                           \
  } while (0)
  auto tile = [&](int t, int b) __attribute__((always_inline)) {
    read_b(b, 0);
    __builtin_amdgcn_sched_barrier(0);
    read_a(b, 0);
    stage(t + 1, RB1, b ^ 1);
    LL_RUN(0, 0);
    read_b(b, 1);
    stage(t + 1, RA1, b ^ 1);
    LL_RUN(0, 1);
    read_a(b, 1);
    stage(t + 2, RA0, b);
    LL_RUN(1, 1);
    stage(t + 2, RB0, b);
    LL_RUN(1, 0);
  };
  const int nsteps = (K + BK - 1) / BK;
  stage(0, RA0, 0); stage(0, RB0, 0); stage(0, RB1, 0); stage(0, RA1, 0);
  stage(1, RA0, 1); stage(1, RB0, 1);
  asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  LL_BARRIER();
  if (wm == 1) LL_BARRIER();        // group 1 runs one barrier interval behind group 0
  for (int t = 0; t < nsteps; t += 2) {
    tile(t, 0);
    tile(t + 1, 1);
  }
  if (wm == 0) LL_BARRIER();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last zero chunks must not land on what the epilogue stages
  LL_BARRIER();
#undef LL_RUN
}

// linear tile index of this workgroup: XCD x (= block % 8) owns a contiguous run of the `total` live tiles; -1: no tile
__device__ __forceinline__ int ll_pos(int total) {
  const int bid = blockIdx.x;
  if (bid >= total) return -1;
  const int q = total >> 3, r = total & 7, xcd = bid & 7, idx = bid >> 3;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

// ------------------------------------------------------------------------------------------------ rows with a label, in order
// order[i] = i-th row with a label, inv[row] = its place or -1, *nvalid; ignored rows get their zero loss here
__global__ __launch_bounds__(1024) void ll_compact_kernel(const int64_t* __restrict__ labels, int rows, int V, int* __restrict__ order,
                                                          int* __restrict__ inv, int* __restrict__ lab, float* __restrict__ row_loss, int* __restrict__ nvalid) {
  __shared__ int cnt[128], pre[128], all;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int r0 = 0; r0 < rows; r0 += 8192) {       // eight labels a thread at a time, loaded together
    int l[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int r = r0 + c * 1024 + tid;
      const int64_t v = r < rows ? labels[r] : -1;
      l[c] = v >= 0 && v < V ? (int)v : -1;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint64_t m = __ballot(l[c] >= 0);
      if (lane == 0) cnt[c * 16 + wave] = __popcll(m);
    }
    __syncthreads();
    if (wave == 0) {                              // 128 (chunk, wave) counts: exclusive prefix sums
      const int a = cnt[2 * lane], b = cnt[2 * lane + 1];
      int t = a + b;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(t, o, 64);
        t += lane >= o ? u : 0;
      }
      pre[2 * lane] = t - a - b;
      pre[2 * lane + 1] = t - b;
      if (lane == 63) all = t;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int r = r0 + c * 1024 + tid;
      const uint64_t m = __ballot(l[c] >= 0);
      if (r < rows) {
        const int at = base + pre[c * 16 + wave] + __popcll(m & ((1ull << lane) - 1ull));
        inv[r] = l[c] >= 0 ? at : -1;
        if (l[c] >= 0) { order[at] = r; lab[at] = l[c]; }
        else row_loss[r] = 0.f;
      }
    }
    base += all;
    __syncthreads();
  }
  if (tid == 0) *nvalid = base;
}

// hp[i] = h[order[i]], columns [d, dp) and rows [nvalid, next multiple of 256) zero; without a list also zk[i] = h_i . W[label_i] (fp32 products, added
// over the lanes' partial sums).  One wave per row.
template <class T>
__global__ __launch_bounds__(256) void ll_pack_kernel(const void* __restrict__ h_, int64_t ldh, const void* __restrict__ w_, int64_t ldw, int d, int dp,
                                                      const int* __restrict__ order, const int* __restrict__ lab, int k, const int* __restrict__ nvalid,
                                                      void* __restrict__ hp_, float* __restrict__ zk, float c, float* __restrict__ eref, int* __restrict__ xtok) {
  typedef typename T::v8 v8;
  typedef typename T::e E;
  const int lane = threadIdx.x & 63, i = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int nv = *nvalid;
  if (i >= (nv + BM - 1) / BM * BM) return;
  E* const dst = (E*)hp_ + (int64_t)i * dp;
  if (i >= nv) {
    if (lane == 0) xtok[i] = -1;
    if (eref && lane == 0) eref[i] = 0.f;
    for (int c = lane * 8; c < dp; c += 512) *(uint4*)(dst + c) = make_uint4(0, 0, 0, 0);
    return;
  }
  const E* const src = (const E*)h_ + order[i] * ldh;
  const E* const wr = (const E*)w_ + lab[i] * ldw;
  float s = 0.f, mass = 0.f;
  for (int c = lane * 8; c < dp; c += 512) {
    const uint4 v = c < d ? *(const uint4*)(src + c) : make_uint4(0, 0, 0, 0);
    *(uint4*)(dst + c) = v;
    if (k == 0 && c < d) {
      const v8 a = __builtin_bit_cast(v8, v), b = *(const v8*)(wr + c);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        s += (float)a[x] * (float)b[x];
        mass += fabsf((float)a[x] * (float)b[x]);
      }
    }
  }
  if (k > 0) return;
  s = ns_wave_sum(s);
  if (lane == 0) { zk[i] = s; xtok[i] = lab[i]; }
  if (!eref) return;
  mass = ns_wave_sum(mass);
  if (lane == 0) eref[i] = ll_label_ref<T>(s, mass, d, c);
}

// zk[i][e] = h_i . W[token e], e = 0 .. k - 1 the teacher's list, e = k the label, and the row's own token (see ll_rows_kernel), the largest of these: a workgroup per row, 16 lanes per entry (256 B of W a step, 16 entries
// side by side; one entry after the other on a wave, 64 entries took 77 us for 1434 rows at d = 512, this 19)
template <class T>
__global__ __launch_bounds__(256) void ll_gather_kernel(const void* __restrict__ hp_, int dp, const void* __restrict__ w_, int64_t ldw, int d, int V,
                                                        const int* __restrict__ order, const int* __restrict__ lab, const int32_t* __restrict__ top_idx,
                                                        int64_t ld_top, int k, const int* __restrict__ nvalid, float* __restrict__ zk, float c1, float* __restrict__ eref,
                                                        int* __restrict__ xtok, float* __restrict__ xz) {
  typedef typename T::v8 v8;
  typedef typename T::e E;
  __shared__ float bz[16], bm[16], lz[2];
  __shared__ int bt[16];
  float top = -INFINITY, top_mass = 0.f;               // this group's largest
  int top_tok = -1;
  const int i = blockIdx.x, l = threadIdx.x & 15;
  if (i >= *nvalid) return;
  const E* const src = (const E*)hp_ + (int64_t)i * dp;
  const int row = order[i];
  for (int e = threadIdx.x >> 4; e <= k; e += 16) {
    const int tok = e == k ? lab[i] : top_idx[row * ld_top + e];
    float s = 0.f, mass = 0.f;
    if (tok >= 0 && tok < V) {
      const E* const wr = (const E*)w_ + tok * ldw;
#pragma unroll 4
      for (int c = l * 8; c < d; c += 128) {
        const v8 a = *(const v8*)(src + c), b = *(const v8*)(wr + c);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          s += (float)a[x] * (float)b[x];
          mass += fabsf((float)a[x] * (float)b[x]);
        }
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) { s += __shfl_xor(s, o, 64); mass += __shfl_xor(mass, o, 64); }
    if (l == 0) zk[(int64_t)i * (k + 1) + e] = s;
    if (l == 0 && e == k) { lz[0] = s; lz[1] = mass; }
    if (tok >= 0 && tok < V && s > top) { top = s; top_mass = mass; top_tok = tok; }
  }
  if (l == 0) { const int g = threadIdx.x >> 4; bz[g] = top; bm[g] = top_mass; bt[g] = top_tok; }
  __syncthreads();
  if (threadIdx.x == 0) {                              // the row's own token: the largest of its list and its label
    float z = lz[0], mass = lz[1];
    int tok = lab[i];
    for (int g = 0; g < 16; ++g)
      if (bz[g] > z) { z = bz[g]; mass = bm[g]; tok = bt[g]; }
    xtok[i] = tok;
    xz[i] = z;
    if (eref) eref[i] = ll_label_ref<T>(z, mass, d, c1);
  }
}

// hT[c][i] = hp[i][c], 64 x 64 tiles through LDS; F (bfloat16): times the row's factor, one rounding
__global__ __launch_bounds__(256) void ll_transpose_kernel(const uint16_t* __restrict__ hp, int dp, const int* __restrict__ nvalid, uint16_t* __restrict__ hT, int ldt,
                                                           const float* __restrict__ F) {
  __shared__ uint16_t t[64][66];
  const int i0 = blockIdx.x * 64, c0 = blockIdx.y * 64;
  if (i0 >= (*nvalid + 63) / 64 * 64) return;
  const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
  for (int r = y; r < 64; r += 4) {
    uint16_t v = hp[(int64_t)(i0 + r) * dp + c0 + x];
    if (F) v = __builtin_bit_cast(uint16_t, (__bf16)((float)__builtin_bit_cast(__bf16, v) * F[i0 + r]));
    t[r][x] = v;
  }
  __syncthreads();
  for (int r = y; r < 64; r += 4) hT[(int64_t)(c0 + r) * ldt + i0 + x] = t[x][r];
}

// ------------------------------------------------------------------------------------------------ the logits' tiles
struct LogitsArgs {
  const void* hp; const void* w; int64_t ldw;
  int dp, d, V, col0, tiles_n, R;        // R: packed rows the buffers are laid out for (a multiple of 256)
  const int* nvalid;
  float c1, c2;                          // log2(e) / temperature of the softmaxes
  float *pm, *p1, *p2;                   // (tiles_n, R): maximum, sum of exp2((z - max) c1), the same with c2
  const float *La, *Lb;                  // (R): base-2 log-sum-exp minus log2 of the weight and of 2^s
  void* G; int ldg;
  float T;
  int row0; float *strip, shift, unshift;   // first packed row; LL_KEEP: (4 tiles_n, R) maxima of the 64-column strips, s and 2^-s
  const int* lab; const float* rk;       // FIX: the label's cell of dz is put right in the staged tile
  const float *eref, *efin;              // REF: (R) the rows' references before and behind the pass
  const int* xtok;                       // the rows' own tokens: no part of the statistics, zero among the kept exponentials
};

// One workgroup per CU walks the tiles of its XCD's run.  The ring never drains: the pieces that a tile's last two K tiles request are the next tile's first
// ones, so a tile has no prologue, and its epilogue runs while they land (one-tile workgroups spent 26 k cycles a tile outside the main loop, which is
// 16 k at d = 512).  Statistics meet in LDS behind the ring.  dz is staged 32 rows x 64 columns at a time in 4 KiB that belong to ONE wave (the two regions
// of ring buffer 1 that hold nothing yet), 16-B chunk c of row r at chunk c ^ (r & 7): no barrier between staging and storing, a wave's own LDS operations
// are in order; its 16 stores are left in flight under the next tile's first K tile, whose waits count them.
constexpr int LL_SIDE = 2 * BUF;                              // behind the ring
constexpr int LL_LOGITS_LDS = LL_SIDE + 3 * 4096 + 2 * 1024;  // statistics: 3 x 4 x 256 floats, two parities of the rows' own tokens; dz: two parities of 4 x 256 row constants (8 KiB)

// MODE LL_STATS: the statistics alone.  LL_KEEP: and 2^(z c1 - e) of every logit in the operands' type, e = the reference of its row (REF) or of its row and
// 64-column strip (minus s for fp16's range), which ll_scale_kernel turns into dz once the rows' sums are known: no logit is formed twice.  LL_GRAD: dz from
// the rows' sums.
enum { LL_STATS, LL_KEEP, LL_GRAD };

// What ll_rows_kernel leaves of a row for its sparse cells, LL_RK floats.  p = 2^(z c1 - E1) I1 with its weight and 2^s, the same with E2, I2 for the second softmax;
// of the row's own token X what the OTHER tokens hold, 1 - p and 1 - q; X; without a list the label's cell, with one (1 - t) - (1 - q) of X.
constexpr int LL_RK = 8;
enum { RK_E1, RK_I1, RK_E2, RK_I2, RK_REST1, RK_REST2, RK_TOKEN, RK_LABEL, RK_SOFT = RK_LABEL };
// SQ (DUAL at T = 2): e^z is the square of e^(z / T), the references' difference an exact power of two: one exponential a logit (1434 rows, d = 512: 123 -> 110 us).
template <class T, int MODE, bool DUAL, bool FIX, bool SQ = false, bool REF = false>
__global__ __launch_bounds__(NTH) void ll_logits_kernel(const LogitsArgs p) {
  constexpr bool GRAD = MODE == LL_GRAD, STORES = MODE != LL_STATS;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef typename T::e E;
  typedef typename T::v8 v8;
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int nv = min(*p.nvalid - p.row0, p.R);
  if (nv <= 0) return;
  const int tiles_m = (nv + BM - 1) / BM, total = tiles_m * p.tiles_n;
  // XCD x (= block % 8) owns a contiguous run of tiles, its workgroups take every nx-th of it
  const int xcd = blockIdx.x & 7, nx = (gridDim.x - xcd + 7) >> 3;
  const int q8 = total >> 3, r8 = total & 7;
  const int x0 = xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8, xn = q8 + (xcd < r8 ? 1 : 0);
  int ti = blockIdx.x >> 3;
  if (ti >= xn) return;
  // eight row tiles by the columns: the 32 workgroups of an XCD that run together read 8 + 4 operand tiles instead of 1 + 32
  auto place = [&](int t, int& tm, int& tn) __attribute__((always_inline)) {
    constexpr int GM = 8;
    const int pos = x0 + t, grp = pos / (GM * p.tiles_n), rem = pos - grp * GM * p.tiles_n;
    const int gm = min(GM, tiles_m - grp * GM);
    tn = rem / gm;
    tm = grp * GM + rem - tn * gm;
  };
  const int ne = ((p.d + BK - 1) / BK + 1) & ~1;              // K tiles, an even number
  uint32_t a_off[2][2], b_off[2][2];
  int my_k[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int rr = 16 * wave + 8 * j + (lane >> 3), ch = (lane & 7) ^ ((rr >> 1) & 7);
    my_k[j] = ch * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      a_off[h][j] = (uint32_t)((((rr >> 6) << 7) + h * 64 + (rr & 63)) * p.dp + ch * 8) * 2u;
      b_off[h][j] = (uint32_t)((((rr >> 5) << 6) + h * 32 + (rr & 31)) * (int)p.ldw + ch * 8) * 2u;
    }
  }
  // operands of the current and the next tile; W's rows end with the vocabulary (a row past it starts behind the resource's last byte)
  auto rsrc_a_of = [&](int tm) __attribute__((always_inline)) { return ll_rsrc((const E*)p.hp + (int64_t)(p.row0 + tm * BM) * p.dp); };
  auto rsrc_b_of = [&](int tn) __attribute__((always_inline)) {
    const int n0 = p.col0 + tn * BN;
    ns_u4v r = ll_rsrc((const E*)p.w + (int64_t)n0 * p.ldw);
    r[2] = (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)min(BN, p.V - n0) * (uint32_t)p.ldw * 2u));
    return r;
  };
  int tm, tn, tm2 = 0, tn2 = 0;
  place(ti, tm, tn);
  bool more = ti + nx < xn;
  if (more) place(ti + nx, tm2, tn2);
  ns_u4v ra = rsrc_a_of(tm), rb = rsrc_b_of(tn), ra2 = rsrc_a_of(tm2), rb2 = rsrc_b_of(tn2);
  const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)smem;
  auto stage = [&](int tt, int region, int buf) __attribute__((always_inline)) {
    const bool nxt = tt >= ne;
    const int k0 = (nxt ? tt - ne : tt) * BK, h = region & 1;
    const bool isb = region >= 2;
    const int klen = nxt && !more ? 0 : (isb ? p.d : p.dp) - k0;
    const ns_u4v rs = isb ? (nxt ? rb2 : rb) : (nxt ? ra2 : ra);
    const uint32_t dst = lds_base + buf * BUF + region * REGION + wave * 2048;
#pragma unroll
    for (int j = 0; j < 2; ++j) ll_dma16(rs, my_k[j] < klen ? (isb ? b_off[h][j] : a_off[h][j]) : OUT, klen > 0 ? k0 * 2 : 0, dst + j * 1024);
  };
  const int fsw = ((lg ^ (l15 >> 1)) & 7) << 4;
  const int a_rd = (wm * 64 + l15) * 128 + fsw, b_rd = (wn * 32 + l15) * 128 + fsw;
  f32x4 acc[2][4][2][2];
  v8 af[4][2], bq[2][2][2];
  auto read_a = [&](int buf, int ah) __attribute__((always_inline)) {
    const char* st = smem + buf * BUF + (ah ? RA1 : RA0) * REGION;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) af[mt][ks] = *(const v8*)(st + ((a_rd ^ (ks << 6)) + mt * 2048));
  };
  auto read_b = [&](int buf, int bh) __attribute__((always_inline)) {
    const char* st = smem + buf * BUF + (bh ? RB1 : RB0) * REGION;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) bq[bh][nt][ks] = *(const v8*)(st + ((b_rd ^ (ks << 6)) + nt * 2048));
  };
  auto mma = [&](int ah, int bh) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) acc[ah][mt][bh][nt] = T::mma(bq[bh][nt][ks], af[mt][ks], acc[ah][mt][bh][nt]);
    __builtin_amdgcn_s_setprio(0);
  };
  // (FIRST, where tiles are stored: the 16 stores of the tile before, 24 with the strips' maxima, lie between the pieces that the first K tile waits for and those it requests)
#define LL_RUN(AH, BH, FIRST)                                               \
  do {                                                                      \
    if (GRAD && (FIRST)) asm volatile("s_waitcnt vmcnt(24)" ::: "memory");  \
    else if (STORES && (FIRST)) asm volatile("s_waitcnt vmcnt(32)" ::: "memory"); \
    else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");                   \
    LL_BARRIER();                                                           \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                      \
    __builtin_amdgcn_sched_barrier(0);                                      \
    mma(AH, BH);                                                            \
    __builtin_amdgcn_sched_barrier(0);                                      \
    LL_BARRIER();                                                           \
  } while (0)
#define LL_KTILE(t, b, FIRST)                               \
  do {                                                      \
    read_b(b, 0);                                           \
    __builtin_amdgcn_sched_barrier(0);                      \
    read_a(b, 0);                                           \
    stage((t) + 1, RB1, (b) ^ 1);                           \
    LL_RUN(0, 0, FIRST);                                    \
    read_b(b, 1);                                           \
    stage((t) + 1, RA1, (b) ^ 1);                           \
    LL_RUN(0, 1, FIRST);                                    \
    read_a(b, 1);                                           \
    stage((t) + 2, RA0, b);                                 \
    LL_RUN(1, 1, FIRST);                                    \
    stage((t) + 2, RB0, b);                                 \
    LL_RUN(1, 0, FIRST);                                    \
  } while (0)
  // row constants of a tile, 256 each: the rows' references and own tokens; of a dz tile La, Lb, the label's column, its cell
  float* const side = (float*)(smem + LL_SIDE);
  auto row_consts = [&](int t, int id, float (&c)[4]) __attribute__((always_inline)) {
    if (REF && id < 256) c[0] = p.eref[p.row0 + t * BM + id];
    if (!GRAD && id < 256) c[1] = __int_as_float(p.xtok[p.row0 + t * BM + id]);
    if (GRAD && id < 256) {
      const int i = t * BM + id;
      c[0] = p.La[i];
      c[1] = DUAL ? p.Lb[i] : 0.f;
      c[2] = c[3] = 0.f;
      if (FIX) {
        c[2] = __int_as_float(i < nv ? p.lab[p.row0 + i] : -1);
        c[3] = i < nv ? p.rk[i * LL_RK + RK_LABEL] : 0.f;
      }
    }
  };
  auto put_consts = [&](int par, int id, const float (&c)[4]) __attribute__((always_inline)) {
    if (REF && id < 256) side[2048 + par * 256 + id] = c[0];      // (one softmax: the third statistic's place is free)
    if (!GRAD && id < 256) side[3072 + par * 256 + id] = c[1];
    if (GRAD && id < 256) {
      side[par * 1024 + id] = c[0];
      if (DUAL) side[par * 1024 + 256 + id] = c[1];
      if (FIX) { side[par * 1024 + 512 + id] = c[2]; side[par * 1024 + 768 + id] = c[3]; }
    }
  };
  // statistics of a finished tile from its four column strips, by the wave group that waits at a tile's start anyway
  auto join = [&](int jm, int jn) __attribute__((always_inline)) {
    const int r = tid & 255;
    float mw[4], mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) { mw[w] = side[w * 256 + r]; mx = fmaxf(mx, mw[w]); }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      s1 += side[1024 + w * 256 + r] * (mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mw[w], p.c1) - ll_ref(mx, p.c1)));
      if (DUAL) s2 += side[2048 + w * 256 + r] * (mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mw[w], p.c2) - ll_ref(mx, p.c2)));
    }
    const int64_t o = (int64_t)jn * p.R + jm * BM + r;
    p.pm[o] = mx;
    p.p1[o] = s1;
    if (DUAL) p.p2[o] = s2;
  };
  int par = 0, jm = -1, jn = 0;
  {
    float c[4];
    row_consts(tm, tid, c);
    put_consts(0, tid, c);
  }
  stage(0, RA0, 0); stage(0, RB0, 0); stage(0, RB1, 0); stage(0, RA1, 0);
  stage(1, RA0, 1); stage(1, RB0, 1);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // (all of it: the first K tile's waits below count a tile's stores, and here are none)
  while (true) {
    LL_BARRIER();
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[a][i][b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (wm == 1) {                    // group 1 runs one barrier interval behind group 0
      if (!GRAD && jm >= 0) join(jm, jn);
      LL_BARRIER();
    }
    for (int t = 0; t < ne; t += 2) {
      int first = t;                  // (laundered: hipcc would peel the first K tile, whose copy spills)
      asm volatile("" : "+s"(first));
      LL_KTILE(t, 0, first == 0);
      LL_KTILE(t + 1, 1, false);
    }
    if (wm == 0) LL_BARRIER();
    const int m0 = tm * BM, n0 = p.col0 + tn * BN;
    // (lane numbers from a laundered copy: hipcc otherwise carries every address of the epilogue through the main loop, and spills)
    int et = tid;
    asm volatile("" : "+v"(et));
    const int el = et & 63, e15 = el & 15, eg = el >> 4;
    const bool edge = n0 + BN > p.V;
    if (edge) {                       // columns past the vocabulary: no part of a row
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n0 + wn * 64 + b * 16 + 4 * eg + r >= p.V) {
#pragma unroll
            for (int ah = 0; ah < 2; ++ah)
#pragma unroll
              for (int mt = 0; mt < 4; ++mt) acc[ah][mt][b >> 1][b & 1][r] = -INFINITY;
          }
    }
    float nc[4];                      // the next tile's row constants
    if (!GRAD && more) row_consts(tm2, et, nc);
    if (!GRAD) {                      // the rows' own tokens: few strips hold one, but most tiles do, and all waves wait for the one whose strip it is
      const int* const own = (const int*)(side + 3072 + par * 256) + wm * 128;
      const int first = n0 + wn * 64;
      const uint64_t hit[2] = {__ballot((unsigned)(own[el] - first) < 64u), __ballot((unsigned)(own[64 + el] - first) < 64u)};
      if (hit[0] | hit[1]) {
#pragma unroll
        for (int ah = 0; ah < 2; ++ah)
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            if (!(hit[ah] >> mt * 16 & 0xFFFF)) continue;
            const int cl = own[ah * 64 + mt * 16 + e15] - first - 4 * eg;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (cl == b * 16 + r) acc[ah][mt][b >> 1][b & 1][r] = -INFINITY;
          }
      }
    }
    if (MODE == LL_STATS) {
      // a el holds 16 of the wave's 64 columns of 8 rows; the row's other lanes are 16 and 32 apart, its other columns in the waves of equal wm
#pragma unroll
      for (int ah = 0; ah < 2; ++ah)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          float mx = -INFINITY;
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[ah][mt][b >> 1][b & 1][r]);
          mx = ll_max4(mx);
          const float e1 = mx == -INFINITY ? 0.f : ll_ref(mx, p.c1), e2 = DUAL ? (mx == -INFINITY ? 0.f : ll_ref(mx, p.c2)) : 0.f;     // (a strip past the vocabulary)
          float s1 = 0.f, s2 = 0.f;
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float z = acc[ah][mt][b >> 1][b & 1][r];
              if (!SQ) s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(z, p.c1, -e1));
              if (DUAL) {
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(z, p.c2, -e2));
                s2 += y;
                if (SQ) s1 = __builtin_fmaf(y, y, s1);
              }
            }
          if (SQ) s1 *= __builtin_amdgcn_exp2f(2.f * e2 - e1);
          s1 = ll_sum4(s1);
          if (DUAL) s2 = ll_sum4(s2);
          if (eg == 0) {
            const int row = wm * 128 + ah * 64 + mt * 16 + e15;
            side[wn * 256 + row] = mx;
            side[1024 + wn * 256 + row] = s1;
            if (DUAL) side[2048 + wn * 256 + row] = s2;
          }
        }
      if (more) put_consts(par ^ 1, et, nc);
      par ^= 1;
    } else if (MODE == LL_KEEP) {
      char* const st = smem + BUF + (wave < 4 ? RA1 : RB1) * REGION + (wave & 3) * 4096;       // this wave's 32 rows x 128 B
      char* const G = (char*)p.G + ((int64_t)(m0 + wm * 128) * p.ldg + tn * BN + wn * 64) * 2;
      float* const strip = p.strip + (int64_t)(tn * 4 + wn) * p.R + m0 + wm * 128;
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) {
        const int ah = qt >> 1;
#pragma unroll
        for (int m2 = 0; m2 < 2; ++m2) {
          const int mt = (qt & 1) * 2 + m2, rl = m2 * 16 + e15, row = wm * 128 + qt * 32 + rl;
          float mx = -INFINITY;
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[ah][mt][b >> 1][b & 1][r]);
          mx = ll_max4(mx);
          // (two softmaxes: what is kept is the one at T, c2 < c1; the sum of the other is taken here from its own exponentials)
          const float ck = DUAL ? p.c2 : p.c1, own = mx == -INFINITY ? 0.f : ll_ref(mx, ck);
          const float e1 = REF ? ll_strip_ref<T>(mx, side[2048 + par * 256 + row], p.c1, p.shift) : own - p.shift;
          const float e2 = DUAL && mx > -INFINITY ? ll_ref(mx, p.c1) : 0.f;
          float s1 = 0.f, s2 = 0.f;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            float g[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float z = acc[ah][mt][b >> 1][b & 1][r];
              g[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(z, ck, -e1));
              s1 += g[r];
              if (SQ) s2 = __builtin_fmaf(g[r], g[r], s2);
              else if (DUAL) s2 += __builtin_amdgcn_exp2f(__builtin_fmaf(z, p.c1, -e2));
            }
            *(ushort4v*)(st + rl * 128 + (((b * 2 + (eg >> 1)) ^ (rl & 7)) << 4) + (eg & 1) * 8) = cvt4<E>(g[0], g[1], g[2], g[3]);
          }
          if (SQ) s2 *= __builtin_amdgcn_exp2f(2.f * e1 - e2);
          s1 = ll_sum4(s1) * (REF ? __builtin_amdgcn_exp2f(fminf(e1 - own, 126.f)) : p.unshift);      // (further below the label than that: a sum of zero)
          if (DUAL) s2 = ll_sum4(s2);
          if (eg == 0) {
            side[wn * 256 + row] = mx;
            side[1024 + wn * 256 + row] = DUAL ? s2 : s1;
            if (DUAL) side[2048 + wn * 256 + row] = s1;
            strip[qt * 32 + rl] = mx;
          }
        }
        if (qt == 0 && more) put_consts(par ^ 1, et, nc);          // (before the first 16-B store: the wait for these loads must not wait for stores)
        asm volatile("" ::: "memory");       // (other lanes' 8-byte writes and these 16-byte reads: the wave's LDS order is all that is needed, hipcc must keep it)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rl = i * 8 + (el >> 3);
          const uint4 v = *(const uint4*)(st + rl * 128 + (((el & 7) ^ (rl & 7)) << 4));
          *(uint4*)(G + (int64_t)(qt * 32 + rl) * p.ldg * 2 + (el & 7) * 16) = v;
        }
        asm volatile("" ::: "memory");
      }
      par ^= 1;
    } else {
      float c[4];
      if (more) row_consts(tm2, et, c);
      char* const st = smem + BUF + (wave < 4 ? RA1 : RB1) * REGION + (wave & 3) * 4096;       // this wave's 32 rows x 128 B
      const float* const rc = side + par * 1024;
      char* const G = (char*)p.G + ((int64_t)(m0 + wm * 128) * p.ldg + tn * BN + wn * 64) * 2;
#pragma unroll
      for (int qt = 0; qt < 4; ++qt) {
        const int ah = qt >> 1;
#pragma unroll
        for (int m2 = 0; m2 < 2; ++m2) {
          const int mt = (qt & 1) * 2 + m2, rl = m2 * 16 + e15, row = wm * 128 + qt * 32 + rl;
          const float la = rc[row], lb = DUAL ? rc[256 + row] : 0.f;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const f32x4 a = acc[ah][mt][b >> 1][b & 1];
            float g[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              g[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(a[r], p.c1, -la));
              if (DUAL) g[r] += __builtin_amdgcn_exp2f(__builtin_fmaf(a[r], p.c2, -lb));
            }
            *(ushort4v*)(st + rl * 128 + (((b * 2 + (eg >> 1)) ^ (rl & 7)) << 4) + (eg & 1) * 8) = cvt4<E>(g[0], g[1], g[2], g[3]);
          }
        }
        if (FIX && el < 32) {
          const int row = wm * 128 + qt * 32 + el, cl = __float_as_int(rc[512 + row]) - (n0 + wn * 64);
          if (cl >= 0 && cl < 64) *(E*)(st + el * 128 + (((cl >> 3) ^ (el & 7)) << 4) + (cl & 7) * 2) = (E)rc[768 + row];
        }
        if (qt == 0 && more) put_consts(par ^ 1, et, c);           // (before the first store: the wait for these loads must not wait for stores)
        asm volatile("" ::: "memory");       // (other lanes' 8-byte writes and these 16-byte reads: the wave's LDS order is all that is needed, hipcc must keep it)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rl = i * 8 + (el >> 3);
          const uint4 v = *(const uint4*)(st + rl * 128 + (((el & 7) ^ (rl & 7)) << 4));
          *(uint4*)(G + (int64_t)(qt * 32 + rl) * p.ldg * 2 + (el & 7) * 16) = v;
        }
        asm volatile("" ::: "memory");
      }
      par ^= 1;
    }
    jm = tm; jn = tn;
    if (!more) break;
    ti += nx;
    tm = tm2; tn = tn2;
    ra = ra2; rb = rb2;
    more = ti + nx < xn;
    if (more) place(ti + nx, tm2, tn2);
    ra2 = rsrc_a_of(tm2); rb2 = rsrc_b_of(tn2);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // this wave's staging reads are done: behind the next barrier its 4 KiB are the ring's again
  }
  if (!GRAD) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    LL_BARRIER();
    if (wm == 1) join(jm, jn);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");              // the last zero chunks land before the workgroup's LDS is given away
#undef LL_KTILE
#undef LL_RUN
}

// dz from what LL_KEEP left, in place: the strip's exponentials times 2^(e - La), one rounding more; a row's label cell (no list) is formed from its own
// logit.  64 rows x 512 columns a workgroup, 16 B per lane; the pass is bound by its bytes (read and written once, mostly in the last-level cache).
// DUAL: what was kept is x = 2^(z c2 - e); softmax(z)'s share is x^T, by its logarithm (a relative rounding of x becomes T of them: T <= 2 only).
template <class T, bool FIX, bool DUAL>
__global__ __launch_bounds__(256) void ll_scale_kernel(const LogitsArgs p) {
  typedef typename T::e E;
  typedef typename T::v8 v8;
  __shared__ float f[8][64], f1[DUAL ? 8 : 1][64];
  __shared__ int lc[64];
  __shared__ float lv[64];
  const int nv = min(*p.nvalid - p.row0, p.R);
  const int i0 = blockIdx.y * 64, t0 = blockIdx.x * 2;
  if (nv <= 0 || i0 >= (nv + BM - 1) / BM * BM) return;
  for (int x = threadIdx.x; x < 512; x += 256) {
    const int sidx = t0 * 4 + (x >> 6), i = i0 + (x & 63);
    if (sidx < p.tiles_n * 4) {
      const float mx = p.strip[(int64_t)sidx * p.R + i];
      const bool none = mx == -INFINITY;      // (past the vocabulary: zeros, whatever the row's logits are.  A factor from no maximum is infinite where they lie low)
      const float e = ll_ref(none ? 0.f : mx, DUAL ? p.c2 : p.c1) - p.shift;
      f[x >> 6][x & 63] = none ? 0.f : __builtin_amdgcn_exp2f(e - (DUAL ? p.Lb[i] : p.La[i]));
      if (DUAL) f1[x >> 6][x & 63] = none ? -INFINITY : e * p.T - p.La[i];
    }
  }
  if (FIX && threadIdx.x < 64) {
    const int i = i0 + threadIdx.x;
    lc[threadIdx.x] = i < nv ? p.lab[p.row0 + i] - t0 * BN : -1;
    lv[threadIdx.x] = i < nv ? p.rk[i * LL_RK + RK_LABEL] : 0.f;
  }
  __syncthreads();
  const int c = (threadIdx.x & 63) * 8, r0 = threadIdx.x >> 6;
  if (t0 * BN + c >= p.tiles_n * BN) return;
  E* const G = (E*)p.G + (int64_t)i0 * p.ldg + t0 * BN + c;
  // (eight loads ahead of the first store: in place, hipcc orders every load behind the store before it)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v8 v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = *(const v8*)(G + (int64_t)(r0 + 4 * (8 * h + x)) * p.ldg);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int r = r0 + 4 * (8 * h + x);
      const float a = f[c >> 6][r], a1 = DUAL ? f1[c >> 6][r] : 0.f;
      const int at = FIX ? lc[r] - c : -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float g = (float)v[x][e] * a;
        if (DUAL) g += __builtin_amdgcn_exp2f(__builtin_fmaf(__builtin_amdgcn_logf((float)v[x][e]), p.T, a1));
        if (FIX && at == e) g = lv[r];
        v[x][e] = (E)g;
      }
      *(v8*)(G + (int64_t)r * p.ldg) = v[x];
    }
  }
}

// REF: the strips that are not kept relative to their row's reference are brought to it, in place.  64 rows x 512 columns a workgroup, a wave per row with such a strip, four
// rows' loads ahead of the first store.  With few of them the launch is all it takes.
template <class T>
__global__ __launch_bounds__(256) void ll_rebase_kernel(const LogitsArgs p) {
  typedef typename T::e E;
  typedef typename T::v8 v8;
  __shared__ float f[8][64];
  __shared__ uint64_t hit[4];
  const int nv = min(*p.nvalid - p.row0, p.R);
  const int i0 = blockIdx.y * 64, t0 = blockIdx.x * 2;
  if (nv <= 0 || i0 >= (nv + BM - 1) / BM * BM) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = i0 + lane;
  const float from = p.eref[p.row0 + i], to = p.efin[i];
  bool any = false;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int st = wave * 2 + x;
    const float mx = t0 * 4 + st < p.tiles_n * 4 ? p.strip[(int64_t)(t0 * 4 + st) * p.R + i] : -INFINITY;
    const float ref = ll_strip_ref<T>(mx, from, p.c1, p.shift);
    const bool moved = mx > -INFINITY && ref != to;          // (a strip past the vocabulary: zeros)
    f[st][lane] = moved ? __builtin_amdgcn_exp2f(ref - to) : 1.f;
    any |= moved;
  }
  const uint64_t mine = __ballot(any);
  if (lane == 0) hit[wave] = mine;
  __syncthreads();
  uint64_t m = hit[0] | hit[1] | hit[2] | hit[3];
  const int c = lane * 8;
  for (int x = 0; x < wave; ++x) m &= m - 1;                // this wave: every fourth of these rows
  E* const G = (E*)p.G + (int64_t)i0 * p.ldg + t0 * BN + c;
  while (m) {
    int r[4];
    v8 v[4];
    float a[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      r[x] = m ? __builtin_ctzll(m) : -1;
      a[x] = r[x] >= 0 ? f[lane >> 3][r[x]] : 1.f;
      if (a[x] != 1.f) v[x] = *(const v8*)(G + (int64_t)r[x] * p.ldg);
#pragma unroll
      for (int b = 0; b < 4; ++b) m &= m - 1;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (a[x] == 1.f) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[x][e] = (E)((float)v[x][e] * a[x]);
      *(v8*)(G + (int64_t)r[x] * p.ldg) = v[x];
    }
  }
}

// ------------------------------------------------------------------------------------------------ rows: log-sum-exp, losses, weights
// How many ways dh's product over one piece of the vocabulary (kt K tiles of 64) is split for `tiles` output tiles: the number that ends soonest when 256
// CUs take (tile, split) pairs in rounds, a pair costing its K tiles and about LL_PAIR more (ring start, fp32 tile to and from its slab).  At most LL_PAIRS
// pairs, eight K tiles each at least.  Depends on sizes and the number of rows with a label alone: the same inputs are added in the same order.
constexpr int LL_PAIRS = 512, LL_PAIR = 6;
__host__ __device__ inline int ll_cost(int tiles, int kt, int s) { return (tiles * s + 255) / 256 * ((kt + s - 1) / s + LL_PAIR); }
__host__ __device__ inline int ll_most_splits(int tiles, int kt) {
  const int a = tiles > 0 ? LL_PAIRS / tiles : 1, b = kt / 8, m = a < b ? a : b;
  return m < 1 ? 1 : m > 1024 ? 1024 : m;
}

// by one workgroup of 256 threads
__device__ __forceinline__ void ll_choose_splits(int nv, int tiles_d, int kt, int* splits) {
  __shared__ unsigned best[4];
  const int tiles = (nv + BM - 1) / BM * tiles_d, most = ll_most_splits(tiles, kt);
  unsigned c = ~0u;
  for (int n = threadIdx.x + 1; n <= most; n += 256) c = min(c, (unsigned)min(ll_cost(tiles, kt, n), 0x1FFFFF) << 11 | (unsigned)n);      // (a tie: the fewest)
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c = min(c, (unsigned)__shfl_xor((int)c, o, 64));
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) *splits = (int)(min(min(best[0], best[1]), min(best[2], best[3])) & 2047);
}

__device__ __forceinline__ float ll_max_or_nan(float a, float b) { return b > a || b != b ? b : a; }

struct RowArgs {
  const float *pm, *p1, *p2;
  int tiles_n, R, k, V, row0;
  int tiles_d, kt; int* splits;
  float c1, c2, invT, w1, w2, lw1, lw2, kd;     // lw*: log2(w* 2^s), -inf for a zero weight; kd: alpha T^2
  int dual, soft_only;                          // one softmax: p1 is at temperature T when only soft targets count
  const int* nvalid; const int *order, *lab;
  const float* z; int64_t ldz;                  // the few-row path's logits (or NULL: the gathered ones)
  float* loss;
  const float* zk; const float* top_vals; const int32_t* top_idx; int64_t ld_top;
  float *La, *Lb, *pk, *row_loss, *packed_loss;
  const int* xtok; const float* xz; float* rk; float up;      // own tokens (many rows) and their logits; LL_RK floats a row; 2^s
  const float* eref; float *efin, *F, head, low, shift;     // REF: the rows' references before and behind the logits' pass, their factors
  float* cl;                                    // p - 1 of the label, where dh's and dW's last steps take it
  int* big_tok; float* big_res; int f16;        // (no list, the label's cell in dz) what the cell's rounding loses: see ll_cells_kernel
};

// 16 threads per row; one workgroup of 1024 threads (the few-row path) also takes the mean.
// A row may be almost certain of a token: p - 1 there is what is left of its gradient, and 1 - p what the OTHER tokens hold.  exp(z - lse) - 1 would have neither the digits
// of 1 - p (lse is rounded at the logits' size: 1 % off at 1 - p = 1e-4) nor, with z gathered and lse from tiles, the same logit on both sides.  So one token a row, its OWN
// (the label, or the largest logit among it and the list), is no part of the statistics: its exponential is added here, from the gathered logit, and 1 - p is the others' share.
template <int NT>
__global__ __launch_bounds__(NT) void ll_rows_kernel(const RowArgs p) {
  constexpr int RB = NT / 16;
  constexpr bool FEW = NT == 1024;
  __shared__ float sm[3][RB][17];
  __shared__ float all[RB];
  __shared__ int xt[FEW ? RB : 1];
  const int nv = min(*p.nvalid - p.row0, p.R), i0 = blockIdx.x * RB;
  if (NT == 256 && blockIdx.x == 0) ll_choose_splits(max(nv, 0), p.tiles_d, p.kt, p.splits);
  if (NT == 256 && (nv <= 0 || i0 >= (nv + BM - 1) / BM * BM)) return;
  const int r_ = threadIdx.x >> 4, q_ = threadIdx.x & 15;
  float xz = -INFINITY;             // the own token's logit
  if (!FEW && i0 + r_ < nv) xz = p.xz[p.row0 + i0 + r_];
  // sixteen partial sums a thread in flight (the first ones under the search for the own token), joined with one exponential each
  const int rs = threadIdx.x & (RB - 1), qs = threadIdx.x / RB;
  float m[16], a[16], b[16];
  auto partials = [&](int t0) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const int64_t o = (int64_t)min(t0 + 16 * x, p.tiles_n - 1) * p.R + i0 + rs;
      m[x] = p.pm[o];
      a[x] = p.p1[o];
      b[x] = p.dual ? p.p2[o] : 0.f;
    }
  };
  partials(qs);
  if (FEW) {
    // few rows: all logits are there, the own token is found here and its tile's others are added up again, without it, in place of the tile's partial sums
    int tok = -1;
    if (r_ < nv) {
      const int lab = p.lab[r_], row = p.order[r_];
      const float* const z = p.z + (int64_t)r_ * p.ldz;
      xz = z[lab];
      tok = lab;
#pragma unroll 4
      for (int e = q_; e < p.k; e += 16) {
        const int t = p.top_idx[row * p.ld_top + e];
        const bool ok = t >= 0 && t < p.V;
        const float v = z[ok ? t : lab];
        if (ok && v > xz) { xz = v; tok = t; }
      }
      if (p.k > 0) {                // (labels alone: nothing waits for the logit here)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
          const float v = __shfl_xor(xz, o, 64);
          const int t = __shfl_xor(tok, o, 64);
          if (v > xz || (v == xz && t > tok)) { xz = v; tok = t; }
        }
      }
    }
    if (q_ == 0) xt[r_] = tok;
    __syncthreads();
  }
  {
    const int r = rs, q = qs;
    const int skip = FEW && xt[r] >= 0 ? xt[r] / BN : -1;
    float mx = -INFINITY, s1 = 0.f, s2 = 0.f;
    for (int t0 = q; t0 < p.tiles_n; t0 += 256) {
      if (t0 != q) partials(t0);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int t = t0 + 16 * x;
        if (t >= p.tiles_n || t == skip) { m[x] = -INFINITY; a[x] = b[x] = 0.f; }
      }
      float nm = mx;
#pragma unroll
      for (int x = 0; x < 16; ++x) nm = fmaxf(nm, m[x]);
      const float n1 = ll_ref(nm, p.c1), n2 = ll_ref(nm, p.c2);
      s1 *= mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mx, p.c1) - n1);      // (a NaN stays one)
      s2 *= mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mx, p.c2) - n2);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        s1 += a[x] * (m[x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(m[x], p.c1) - n1));
        if (p.dual) s2 += b[x] * (m[x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(m[x], p.c2) - n2));
      }
      mx = nm;
    }
    sm[0][r][q] = mx; sm[1][r][q] = s1; sm[2][r][q] = s2;
  }
  __syncthreads();
  const int r = r_, q = q_, i = i0 + r;
  float mo = sm[0][r][q], s1 = sm[1][r][q], s2 = sm[2][r][q];      // of the others, relative to 2^ref(mo)
  if (FEW && i < nv) {
    const int tok = xt[r], c0 = tok / BN * BN + q * 16;
    const float* const z = p.z + (int64_t)i * p.ldz + c0;
    float v[16], m = mo;
#pragma unroll
    for (int x = 0; x < 16; x += 4) *(f32x4*)&v[x] = *(const f32x4*)(z + x);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      if (c0 + x >= p.V || c0 + x == tok) v[x] = -INFINITY;
      m = fmaxf(m, v[x]);
    }
    const float n1 = m == -INFINITY ? 0.f : ll_ref(m, p.c1), n2 = m == -INFINITY ? 0.f : ll_ref(m, p.c2);
    s1 *= mo == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mo, p.c1) - n1);
    s2 *= mo == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mo, p.c2) - n2);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(v[x], p.c1, -n1));
      if (p.dual) s2 += __builtin_amdgcn_exp2f(__builtin_fmaf(v[x], p.c2, -n2));
    }
    mo = m;
  }
  float mx = mo;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  const float others = mx;          // the largest logit but the own token's
  mx = fmaxf(mx, xz);
  const float e1 = ll_ref(mx, p.c1), e2 = ll_ref(mx, p.c2);      // the sums are relative to 2^e1, 2^e2
  s1 *= mo == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mo, p.c1) - e1);
  s2 *= mo == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(mo, p.c2) - e2);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) { s1 += __shfl_xor(s1, o, 64); s2 += __shfl_xor(s2, o, 64); }
  const float o1 = s1, o2 = s2;
  s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(xz, p.c1, -e1));
  s2 += __builtin_amdgcn_exp2f(__builtin_fmaf(xz, p.c2, -e2));
  const float rest1 = o1 / s1, rest2 = p.dual ? o2 / s2 : rest1;      // (one softmax: it is the one at T)
  const bool live = i < nv;
  float loss = 0.f;
  if (!live) {                      // padding rows of the last tile: no probability
    if (q == 0) {
      p.La[i] = INFINITY;
      if (p.Lb) p.Lb[i] = INFINITY;
      if (p.eref) { p.efin[i] = 0.f; p.F[i] = 0.f; }
    }
    if (NT == 256) return;
  }
  if (live) {
  const int pi = p.row0 + i, row = p.order[pi];
  auto logit = [&](int e, int tok) __attribute__((always_inline)) { return p.z ? p.z[(int64_t)i * p.ldz + tok] : p.zk[(int64_t)pi * (p.k + 1) + e]; };
  bool soft = false;
  float soft_rest = 0.f;
  if (p.k > 0) {
    // the teacher's distribution over the entries that name a token; a list without any leaves the hard label alone
    const float* const tv = p.top_vals + row * p.ld_top;
    const int32_t* const ti = p.top_idx + row * p.ld_top;
    float tm = -INFINITY;
    // (value and token loaded side by side, four entries in flight: a value behind its token's test took a memory latency more per entry)
#pragma unroll 4
    for (int e = q; e < p.k; e += 16) {
      const int t = ti[e];
      const float v = tv[e] * p.invT;
      tm = t >= 0 && t < p.V ? ll_max_or_nan(tm, v) : tm;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) tm = ll_max_or_nan(tm, __shfl_xor(tm, o, 64));
    soft = tm != -INFINITY;               // (a NaN or +inf that an entry holds shows in the row's loss)
    float ts = 0.f;
#pragma unroll 4
    for (int e = q; e < p.k; e += 16) {
      const int t = ti[e];
      const float v = tv[e] * p.invT;
      ts += soft && t >= 0 && t < p.V ? expf(v - tm) : 0.f;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) ts += __shfl_xor(ts, o, 64);
    const float lt = logf(ts), inv = 1.f / ts;
    const float ls = log2f(p.dual ? s2 : s1);     // (one softmax: it is the one at T)
    float kl = 0.f, lr = 0.f;
    const int x = FEW ? xt[r] : p.xtok[pi];
#pragma unroll 4
    for (int e = q; e < p.k; e += 16) {
      float pr = 0.f;
      const int t = ti[e];
      const float lp = tv[e] * p.invT - tm;
      const bool ok = soft && t >= 0 && t < p.V;
      const float z = logit(e, ok ? t : 0);
      if (ok) {
        pr = expf(lp) * inv;
        if (pr != 0.f) kl += pr * ((lp - lt) - (__builtin_fmaf(z, p.c2, -e2) - ls) * LN2);
      }
      p.pk[(int64_t)pi * p.k + e] = pr;
      lr += t == x ? 0.f : pr;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) { kl += __shfl_xor(kl, o, 64); lr += __shfl_xor(lr, o, 64); }
    if (soft) { loss += p.kd * kl; soft_rest = lr - rest2; }
  }
  if (q == 0) {
    if (!p.soft_only) loss -= p.w1 * (__builtin_fmaf(logit(p.k, p.lab[pi]), p.c1, -e1) - log2f(s1)) * LN2;      // (lse - z in units of ln 2)
    const float l1 = e1 + log2f(s1);
    if (p.dual) {
      p.La[i] = l1 - p.lw1;
      p.Lb[i] = soft ? e2 + log2f(s2) - p.lw2 : INFINITY;
    } else if (p.k > 0) {
      // one softmax carries both weights (T = 1), or the soft weight alone
      const float w = (p.soft_only ? 0.f : p.w1) + (soft ? p.w2 : 0.f);
      p.La[i] = w > 0.f ? l1 - (p.lw1 + log2f(w)) : INFINITY;      // (lw1 is log2(2^s) here)
    } else {
      p.La[i] = l1 - p.lw1;
    }
    if (p.eref) {
      const float a = p.eref[pi];
      const bool keeps = others * p.c1 <= a + p.head && log2f(o1) + e1 >= a + p.low;
      const float e = keeps ? a : ll_ref(others == -INFINITY ? mx : others, p.c1) - p.shift;
      p.efin[i] = e;
      p.F[i] = __builtin_amdgcn_exp2f(e - p.La[i] - p.shift);      // (La is for cells times 2^shift)
      if (p.cl) p.cl[i] = -rest1;
    }
    if (p.rk) {
      const float i1 = (p.dual || p.k == 0 ? p.w1 : (p.soft_only ? 0.f : p.w1) + (soft ? p.w2 : 0.f)) * p.up / s1;
      f32x4* const rk = (f32x4*)(p.rk + (int64_t)i * LL_RK);
      rk[0] = f32x4{e1, i1, e2, p.dual && soft ? p.w2 * p.up / s2 : 0.f};
      const int own = rest1 < 0.5f || rest2 < 0.5f ? (FEW ? xt[r] : p.xtok[pi]) : -1;      // (a row that is certain of nothing: p itself has the digits)
      rk[1] = f32x4{rest1, rest2, __int_as_float(own), p.k == 0 ? -p.w1 * p.up * rest1 : soft_rest};
    }
    if (p.big_tok) {
      const float v = -p.w1 * p.up * rest1;
      p.big_tok[2 * pi] = p.lab[pi];
      p.big_tok[2 * pi + 1] = -1;
      p.big_res[2 * pi] = v - (p.f16 ? (float)(half_t)v : (float)(__bf16)v);
      p.big_res[2 * pi + 1] = 0.f;
    }
    p.row_loss[row] = loss;
    if (NT == 256) p.packed_loss[pi] = loss;
  }
  }
  if (NT == 1024) {
    if (q == 0) all[r] = live ? loss : 0.f;
    __syncthreads();
    if (threadIdx.x < 64) {
      const float s = ns_wave_sum(all[threadIdx.x]);
      if (threadIdx.x == 0) *p.loss = s / (float)max(nv, 1);
    }
  }
}

// the loss: a launch of its own where no dh is asked for, else a workgroup of the kernel that writes dh
template <int NT> __device__ __forceinline__ void ll_mean(const float* __restrict__ packed_loss, int nv, float* __restrict__ loss) {
  __shared__ float sh[NT / 64];
  float s = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < nv; i += NT) s += packed_loss[i];
  s = ns_wave_sum(s);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    for (int w = 0; w < NT / 64; ++w) s += sh[w];
    *loss = s / (float)max(nv, 1);
  }
}
__global__ __launch_bounds__(1024) void ll_mean_kernel(const float* __restrict__ packed_loss, const int* __restrict__ nvalid, float* __restrict__ loss) {
  ll_mean<1024>(packed_loss, *nvalid, loss);
}

// a cell of dz at a token that the label or the list names (soft: the list's probability of it; own: the row is certain of it, and p - 1 = -(1 - p), q - t = (1 - t) - (1 - q))
struct RowK { f32x4 lo, hi; };
__device__ __forceinline__ RowK ll_row_k(const float* rk) { return {*(const f32x4*)rk, *(const f32x4*)(rk + 4)}; }
__device__ __forceinline__ float ll_sparse_cell(const RowK& k, float z, float c1, float c2, float w1s, float w2s, float soft, bool own, bool label) {
  static_assert(RK_E1 == 0 && RK_I1 == 1 && RK_E2 == 2 && RK_I2 == 3 && RK_REST1 == 4 && RK_SOFT == 7, "ll_rows_kernel writes them in this order");
  if (own) return (label ? -w1s * k.hi[0] : w1s * (1.f - k.hi[0])) + (w2s > 0.f ? w2s * k.hi[3] : 0.f);
  float v = __builtin_amdgcn_exp2f(__builtin_fmaf(z, c1, -k.lo[0])) * k.lo[1];
  if (k.lo[3] > 0.f) v = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(z, c2, -k.lo[2])), k.lo[3], v);
  return v - w2s * soft - (label ? w1s : 0.f);
}

// the sparse cells of dz in one piece: one wave per row, each token written once whatever number of entries name it.
// A row's gradient is mostly its one or two largest cells, whose rounding would be an error of all of it (1.5 times the result's own where few rows average it out):
// what the two largest lose goes to big_tok / big_res, and dh's and dW's last steps add it in fp32 (fp16, 1434 rows with lists, dh and dW: 2.6e-4 -> 2.1e-4 off, the
// result's own rounding, for 15 us of 398).
template <class E>
__global__ __launch_bounds__(256) void ll_cells_kernel(const int* __restrict__ nvalid, int row0, int R, const int* __restrict__ order, const int* __restrict__ lab,
                                                       const int32_t* __restrict__ top_idx, int64_t ld_top, int k, const float* __restrict__ zk,
                                                       const float* __restrict__ pk, const float* __restrict__ La, const float* __restrict__ rk, float c1, float c2,
                                                       float w1s, float w2s, int col0, int cols, int V, E* __restrict__ G, int ldg, const float* __restrict__ efin,
                                                       int* __restrict__ big_tok, float* __restrict__ big_res) {
  __shared__ __attribute__((aligned(16))) int sidx[4][LL_MAX_K + 4];
  __shared__ __attribute__((aligned(16))) float sp[4][LL_MAX_K + 4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = blockIdx.x * 4 + wave;
  const int nv = min(*nvalid - row0, R), pi = row0 + i;
  const bool live = i < nv;
  if (live) {
    const int row = order[pi];
    for (int e = lane; e < k + 4; e += 64) {       // (k + 1 entries and none behind them)
      const int t = e == k ? lab[pi] : e < k ? top_idx[row * ld_top + e] : -1;
      sidx[wave][e] = t >= 0 && t < V ? t : -1;
      sp[wave][e] = e < k ? pk[(int64_t)pi * k + e] : 0.f;
    }
  }
  __syncthreads();
  if (!live) return;
  // (efin: cells relative to the row's factor; one of zero leaves none)
  const float la = La[i], up = efin ? (la < INFINITY ? __builtin_amdgcn_exp2f(la - efin[i]) : 0.f) : 1.f;
  const RowK kk = ll_row_k(rk + (int64_t)i * LL_RK);
  const int own = __float_as_int(kk.hi[RK_TOKEN - 4]);
  float m1 = 0.f, m2 = 0.f, r1 = 0.f, r2 = 0.f;             // this lane's two largest
  int t1 = -1, t2 = -1;
  for (int e = lane; e <= k; e += 64) {
    const int t = sidx[wave][e], c = t - col0;
    const bool in = c >= 0 && c < cols;
    if (t < 0 || (!in && col0 > 0)) continue;               // (the first piece's launch looks at all of a row's cells)
    float soft = 0.f;
    bool first = true;
#pragma unroll 4
    for (int o = 0; o < k; o += 4) {                        // (sp[k] is zero, and entry k comes no earlier than any)
      const int4 s = *(const int4*)&sidx[wave][o];
      const f32x4 q = *(const f32x4*)&sp[wave][o];
      soft += (s.x == t ? q[0] : 0.f) + (s.y == t ? q[1] : 0.f) + (s.z == t ? q[2] : 0.f) + (s.w == t ? q[3] : 0.f);
      first = first && !((s.x == t && o < e) || (s.y == t && o + 1 < e) || (s.z == t && o + 2 < e) || (s.w == t && o + 3 < e));
    }
    if (!first) continue;                                   // an earlier entry of the list names the same token: that one writes
    const float v = up * ll_sparse_cell(kk, zk[(int64_t)pi * (k + 1) + e], c1, c2, w1s, w2s, soft, t == own, t == lab[pi]);
    if (in) G[(int64_t)i * ldg + c] = (E)v;
    const float m = fabsf(v), res = v - (float)(E)v;
    if (m > m1) { m2 = m1; t2 = t1; r2 = r1; m1 = m; t1 = t; r1 = res; }
    else if (m > m2) { m2 = m; t2 = t; r2 = res; }
  }
  if (col0 > 0) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float m = ns_wave_max(m1);
    const uint64_t who = __ballot(m1 == m && m1 > 0.f);
    if (who == 0) {
      if (lane == 0) { big_tok[2 * pi + j] = -1; big_res[2 * pi + j] = 0.f; }
    } else if (lane == __builtin_ctzll(who)) {
      big_tok[2 * pi + j] = t1;
      big_res[2 * pi + j] = r1;
      m1 = m2; t1 = t2; r1 = r2;
    }
  }
}

// ------------------------------------------------------------------------------------------------ dh += dz W,  dW = dz^T h
struct DhArgs {
  const void* G; const void* w; int64_t ldw;
  int ldg, col0, cols, V, d, kt, add, row0, R;
  const int *nvalid, *splits;
  float* slab;                      // (splits, tiles, 256, 256)
};

template <class T>
__global__ __launch_bounds__(NTH) void ll_dh_kernel(const DhArgs p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef typename T::e E;
  const int nv = min(*p.nvalid - p.row0, p.R);
  if (nv <= 0) return;
  const int tiles_m = (nv + BM - 1) / BM, tiles_d = (p.d + BN - 1) / BN;
  const int tiles = tiles_m * tiles_d, splits = *p.splits;
  const int pos = ll_pos(tiles * splits);
  if (pos < 0) return;
  const int split = pos / tiles, t = pos - split * tiles;
  const int tm = t / tiles_d, td = t - tm * tiles_d;
  const int m0 = tm * BM, n0 = td * BN;
  const int chunk = (p.kt + splits - 1) / splits * BK, k0 = split * chunk, kn = min(chunk, p.cols - k0);          // (a split past the end leaves its zeros)
  f32x4 acc[2][4][2][2];
  ll_tile<T, true, false>(acc, smem, (const E*)p.G + (int64_t)m0 * p.ldg + k0, p.ldg, kn,
                          (const E*)p.w + (int64_t)(p.col0 + k0) * p.ldw + n0, (int)p.ldw, min(kn, p.V - p.col0 - k0), min(BN, p.d - n0), max(kn, 0));
  const int lane = threadIdx.x & 63, l15 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  float* const out = p.slab + (int64_t)pos * (BM * BN);
  // eight 16-B loads in flight before the first addition (a load, an addition and a store at a time cost a memory latency each)
#pragma unroll
  for (int ah = 0; ah < 2; ++ah)
#pragma unroll
    for (int mp = 0; mp < 4; mp += 2) {
      f32x4 old[2][4];
      if (p.add) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int rl = wm * 128 + ah * 64 + (mp + m) * 16 + l15, cl = wn * 64 + b * 16 + 4 * lg;
            old[m][b] = *(const f32x4*)(out + rl * BN + cl);
          }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int rl = wm * 128 + ah * 64 + (mp + m) * 16 + l15, cl = wn * 64 + b * 16 + 4 * lg;
          f32x4 v = acc[ah][mp + m][b >> 1][b & 1];
          if (p.add) v += old[m][b];
          *(f32x4*)(out + rl * BN + cl) = v;
        }
    }
}

// dh[row] = g 2^-s sum of the slabs (in their order), zero for a row without a label.  A workgroup takes 64 columns of a row with 16 threads of 4 columns,
// and 16 groups of slabs side by side: with one token and 203 slabs a single chain of loads took 28 us
// (R > 0: slabs of (R, d) from the few-row path; R = 0: slabs of 256 x 256 tiles, their number read from splits_dev.)
template <class E>
__global__ __launch_bounds__(256) void ll_dh_out_kernel(const float* __restrict__ slab, int groups, int splits, const int* __restrict__ splits_dev, int R, int row0, int chunk, int d, int rows, const int* __restrict__ inv,
                                                        const int* __restrict__ nvalid, const float* __restrict__ loss_scale, float unscale, E* __restrict__ dh, int64_t lddh,
                                                        const float* __restrict__ packed_loss, float* __restrict__ loss, const float* __restrict__ F, const E* __restrict__ w,
                                                        int64_t ldw, const int* __restrict__ lab, const float* __restrict__ cl, const int* __restrict__ big_tok, const float* __restrict__ big_res) {
  if (loss && blockIdx.x == gridDim.x - 1) {      // one workgroup more: the mean of the row losses
    ll_mean<256>(packed_loss, *nvalid, loss);
    return;
  }
  typedef E e4 __attribute__((ext_vector_type(4)));
  __shared__ f32x4 sm[16][16];
  // `groups` slab groups; the rest of the 16 lanes-of-16 take further column blocks
  const int sub = threadIdx.x >> 4, g = sub & (groups - 1), blk = sub / groups;
  const int per = (d + 63) / 64, nblk = 16 / groups;
  const int64_t x = (int64_t)blockIdx.x * nblk + blk;
  const int row = (int)(x / per), c = (int)(x - (int64_t)row * per) * 64 + (threadIdx.x & 15) * 4;
  const bool in = row < rows && c < d;
  const int pi = in ? inv[row] : -1, i = pi >= row0 && pi - row0 < chunk ? pi - row0 : -1;      // a chunk writes its own rows, the first one the ignored ones
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  if (i >= 0) {
    if (splits_dev) splits = *splits_dev;
    const int per_g = (splits + groups - 1) / groups, s1 = min(splits, (g + 1) * per_g);
    const int tiles_d = (d + BN - 1) / BN, tiles = (min(*nvalid - row0, chunk) + BM - 1) / BM * tiles_d;
    const int64_t at = R > 0 ? (int64_t)i * d + c : ((int64_t)(i / BM * tiles_d + c / BN) * BM + i % BM) * BN + c % BN;
    const int64_t step = R > 0 ? (int64_t)R * d : (int64_t)tiles * BM * BN;
    if (R > 0 && 2 * *nvalid <= R) {             // (rows that are in two parts: R / 2 further is what the first part's rounding lost)
#pragma unroll 4
      for (int s = g * per_g; s < s1; ++s) a += *(const f32x4*)(slab + s * step + at) + *(const f32x4*)(slab + s * step + at + (int64_t)(R / 2) * d);
    } else {
#pragma unroll 4
      for (int s = g * per_g; s < s1; ++s) a += *(const f32x4*)(slab + s * step + at);
    }
  }
  if (groups > 1) {
    sm[sub][threadIdx.x & 15] = a;
    __syncthreads();
    if (g == 0)
      for (int o = 1; o < groups; ++o) a += sm[sub + o][threadIdx.x & 15];
  }
  if (!in || g != 0 || (pi >= 0 ? i < 0 : row0 > 0)) return;
  const float gs = (loss_scale ? *loss_scale : 1.f) / (float)max(*nvalid, 1);
  if (i >= 0) {
    if (big_tok) {                                // what the two largest cells' rounding lost
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = big_tok[2 * pi + j];
        if (t < 0) continue;
        const float r = big_res[2 * pi + j];
        const e4 l = *(const e4*)(w + t * ldw + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = __builtin_fmaf(r, (float)l[e], a[e]);
      }
    }
    a *= F ? F[i] : unscale;
    if (cl) {                                     // the label's part, which is not in dz then
      const e4 l = *(const e4*)(w + lab[pi] * ldw + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] = __builtin_fmaf(cl[i], (float)l[e], a[e]);
    }
  }
  e4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (E)(i < 0 ? 0.f : a[e] * gs);
  *(e4*)(dh + row * lddh + c) = o;
}
template <class E> void launch_dh_out(const float* slab, int groups, int splits, const int* splits_dev, int R, int row0, int chunk, int d, int rows, const int* inv, const int* nvalid, const float* loss_scale, float unscale, E* dh,
                                      int64_t lddh, const float* packed_loss, float* loss, const float* F, const E* w, int64_t ldw, const int* lab, const float* cl, const int* big_tok, const float* big_res, hipStream_t st) {
  const int nblk = 16 / groups;
  const int64_t items = (int64_t)rows * ((d + 63) / 64);
  if (items == 0 && !loss) return;               // (no rows: nothing to write)
  hipLaunchKernelGGL(ll_dh_out_kernel<E>, dim3((unsigned)((items + nblk - 1) / nblk) + (loss ? 1 : 0)), dim3(256), 0, st, slab, groups, splits, splits_dev, R, row0, chunk, d, rows, inv, nvalid,
                     loss_scale, unscale, dh, lddh, packed_loss, loss, F, w, ldw, lab, cl, big_tok, big_res);
}

struct DwArgs {
  const void* hT; int ldt;
  const void* G; int ldg, col0, tiles_v, V, d, row0, R;
  const int* nvalid; const float* loss_scale;
  float unscale;
  void* dw; int64_t lddw; int f32, add;
  const void* hp; int dp;
  const int* tok; const float* coef; int per;                   // (2^per a packed row) tokens and coefficients of h that dz does not hold: the labels' cells, or what the largest cells' rounding lost
};

// What dz does not hold of dW's tile, in fp32: the labels' part where h's copy is rounded with the rows' factors (a token's row of dW is mostly its labels' h), else what the
// largest cells' rounding lost.  Entries whose token is one of the tile's 256 are listed in order, 4096 at a time, and each adds coefficient x h to its token's
// accumulators (bf16, no list: dW 2.8e-3 -> 1.7e-3 off, its own rounding, for 12 us of 382 at 1844 rows, d = 512).
constexpr int LL_LIST = 4096;
template <class T>
__device__ __forceinline__ void ll_add_entries(f32x4 (&acc)[2][4][2][2], char* smem, const DwArgs& p, int entries, int v0, int m0) {
  typedef typename T::e E;
  typedef E e4 __attribute__((ext_vector_type(4)));
  int2* const list = (int2*)smem;
  int* const cnt = (int*)(smem + LL_LIST * 8);            // 64 counts, 64 prefixes, the sum
  char* const rows = (char*)(cnt + 132);
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));                             // (no address of this part is carried through the main loop, where there is no register for it)
  const int lane = tid & 63, l15 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 2, wn = wave & 3;
  for (int base = 0; base < entries; base += LL_LIST) {
    int t[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int i = base + x * NTH + tid;
      t[x] = i < entries ? p.tok[i] : -1;
      t[x] = t[x] < 0 ? -1 : t[x] - v0;
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint64_t m = __ballot(t[x] >= 0 && t[x] < BN);
      if (lane == 0) cnt[x * 8 + wave] = __popcll(m);
    }
    __syncthreads();
    if (wave == 0) {
      const int own = cnt[lane];
      int sum = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(sum, o, 64);
        sum += lane >= o ? u : 0;
      }
      cnt[64 + lane] = sum - own;
      if (lane == 63) cnt[128] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const bool hit = t[x] >= 0 && t[x] < BN;
      const uint64_t m = __ballot(hit);
      if (hit) list[cnt[64 + x * 8 + wave] + __popcll(m & ((1ull << lane) - 1ull))] = make_int2(base + x * NTH + tid, t[x]);
    }
    __syncthreads();
    // 64 rows of h at a time through LDS (their loads in flight together, no registers), then a wave takes the rows whose token is one of its 64
    const int n = cnt[128];
    for (int e0 = 0; e0 < n; e0 += 64) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int e = (tid >> 5) + 16 * x, col = (tid & 31) * 8;
        if (e0 + e < n && m0 + col < p.dp) *(uint4*)(rows + e * LDH + col * 2) = *(const uint4*)((const E*)p.hp + (int64_t)(list[e0 + e].x >> p.per) * p.dp + m0 + col);
      }
      const int2 it = e0 + lane < n ? list[e0 + lane] : make_int2(0, -1);
      const float cl = it.y >= 0 ? p.coef[it.x] : 0.f;
      uint64_t m = __ballot(it.y >= 0 && it.y >> 6 == wn);
      __syncthreads();
      while (m) {
        const int e = __builtin_ctzll(m), tok = __builtin_amdgcn_readlane(it.y, e);
        const float c = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(cl), e));
        m &= m - 1;
#pragma unroll
        for (int ah = 0; ah < 2; ++ah) {
          f32x4 a[4];
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            const int col = wm * 128 + ah * 64 + mt * 16 + 4 * lg;
            a[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (l15 == (tok & 15) && m0 + col < p.dp) {
              const e4 v = *(const e4*)(rows + e * LDH + col * 2);
#pragma unroll
              for (int r = 0; r < 4; ++r) a[mt][r] = c * (float)v[r];
            }
          }
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if ((tok >> 4 & 3) == b) {
#pragma unroll
              for (int mt = 0; mt < 4; ++mt) acc[ah][mt][b >> 1][b & 1] += a[mt];
            }
        }
      }
      __syncthreads();
    }
  }
  __syncthreads();                                          // (a batch of no entries ends with every wave's read of its count: the caller stages over it)
}

template <class T>
__global__ __launch_bounds__(NTH) void ll_dw_kernel(const DwArgs p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef typename T::e E;
  const int tiles_d = (p.d + BM - 1) / BM;
  const int pos = ll_pos(tiles_d * p.tiles_v);
  if (pos < 0) return;
  const int tv = pos / tiles_d, td = pos - tv * tiles_d;
  const int m0 = td * BM, n0 = tv * BN;                    // columns of h, columns of dz (= rows of W)
  const int nv = *p.nvalid, K = max(min(nv - p.row0, p.R) + BK - 1, 0) / BK * BK;
  f32x4 acc[2][4][2][2];
  ll_tile<T, true, true>(acc, smem, (const E*)p.hT + (int64_t)m0 * p.ldt + p.row0, p.ldt, K, (const E*)p.G + n0, p.ldg, K, BN, K);
  const float gs = (p.loss_scale ? *p.loss_scale : 1.f) / (float)max(nv, 1) * p.unscale;
  const int tid = threadIdx.x, lane = tid & 63, l15 = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  // a lane owns 4 consecutive columns of h (m) of one row of W (n)
  const int v0 = p.col0 + n0;
  ll_add_entries<T>(acc, smem, p, nv << p.per, v0, m0);
  if (p.f32) {
    float* const out = (float*)p.dw + (int64_t)v0 * p.lddw + m0;
#pragma unroll
    for (int ah = 0; ah < 2; ++ah)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int cl = wm * 128 + ah * 64 + mt * 16 + 4 * lg, rl = wn * 64 + b * 16 + l15;
          if (m0 + cl >= p.d || v0 + rl >= p.V) continue;
          f32x4* const at = (f32x4*)(out + (int64_t)rl * p.lddw + cl);
          f32x4 v = acc[ah][mt][b >> 1][b & 1] * gs;
          if (p.add) v += *at;
          *at = v;
        }
    return;
  }
  // 16-bit: staged as rows of W, stored (or added to what is there, in fp32) 512 B a row
#pragma unroll
  for (int ah = 0; ah < 2; ++ah)
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int cl = wm * 128 + ah * 64 + mt * 16 + 4 * lg, rl = wn * 64 + b * 16 + l15;
        const f32x4 v = acc[ah][mt][b >> 1][b & 1] * gs;
        *(ushort4v*)(smem + rl * LDH + cl * 2) = cvt4<E>(v[0], v[1], v[2], v[3]);
      }
  __syncthreads();
  const int cg = tid & 31;
  if (m0 + cg * 8 >= p.d) return;
  typedef typename T::v8 v8;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int rl = (tid >> 5) + 16 * i;
    if (v0 + rl >= p.V) continue;
    *(v8*)((E*)p.dw + (int64_t)(v0 + rl) * p.lddw + m0 + cg * 8) = *(const v8*)(smem + rl * LDH + cg * 16);
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to LL_FEW_ROWS rows: the time is W's bytes, read once for the logits and once more for dh (dW is written once).  No 256-row tiles, no packing, and
// the logits of so few rows (N V fp32, 13 MB at 64) ARE kept, in the workspace: nothing is formed twice.
//   ll_few_logits  a workgroup takes 256 rows of W, a wave 32 of them, 64 columns at a time by LDS-DMA, three chunks in flight
//   ll_rows        as for many rows, one workgroup for all of them, and the mean
//   ll_few_grad    a workgroup takes 256 tokens: dz of those (rows x 256, in LDS, sparse cells put right there), then 64 columns of W at a time by LDS-DMA,
//                  three chunks in flight: dh's part of these tokens, and the tokens' rows of dW
// Rows with a label are found by every workgroup itself: one ballot over at most 64 labels.
constexpr int LL_FEW_ROWS = 64;

// this wave's view: number of rows with a label; src = original row of packed row `lane` (or -1)
__device__ __forceinline__ int few_rows(const int64_t* labels, int rows, int V, int lane, int& src) {
  const int64_t l = lane < rows ? labels[lane] : -1;
  const bool ok = l >= 0 && l < V;
  const uint64_t m = __ballot(ok);
  const int n = __popcll(m);
  // the lane-th set bit of m: binary search over prefix counts
  int pos = 0;
#pragma unroll
  for (int b = 32; b > 0; b >>= 1) {
    const uint64_t low = pos + b >= 64 ? m : m & ((1ull << (pos + b)) - 1ull);
    if (__popcll(low) <= lane) pos += b;
  }
  src = lane < n ? pos : -1;
  return n;
}

struct FewArgs {
  const void* h; int64_t ldh; const void* w; int64_t ldw;
  const int64_t* labels;
  int rows, d, V, tiles_n;
  float c1, c2;
  float* z; int64_t ldz;            // (16 MT, tiles_n 256)
  float *pm, *p1, *p2; int R;       // (tiles_n, R)
  int *order, *inv, *lab, *nvalid; float* row_loss;
  // gradient
  const float *La, *Lb, *pk, *rk; const int32_t* top_idx; int64_t ld_top; int k;
  float w1s, w2s, unscale;
  const float* loss_scale;
  float* slab;                      // (tiles_n, 16 MT, d)
  void* dw; int64_t lddw; int f32, add, dh;
};

constexpr int FW_BYTES = 256 * 128;          // a chunk of W: 256 tokens x 64 columns
constexpr int FH_BYTES = 64 * 128;           // a chunk of h: 64 rows x 64 columns
constexpr int FL_LDS = 3 * (FW_BYTES + FH_BYTES);

template <class T, int MT, bool DUAL>
__global__ __launch_bounds__(512) void ll_few_logits_kernel(const FewArgs p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef typename T::e E;
  typedef typename T::v8 v8;
  __shared__ float sm[3][8][16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, lg = lane >> 4;
  int src;
  const int nv = few_rows(p.labels, p.rows, p.V, lane, src);
  if (blockIdx.x == 0 && wave == 0) {
    if (lane < p.rows) {
      const int64_t l = p.labels[lane];
      const bool ok = l >= 0 && l < p.V;
      const uint64_t m = __ballot(ok);
      p.inv[lane] = ok ? __popcll(m & ((1ull << lane) - 1ull)) : -1;
      if (!ok) p.row_loss[lane] = 0.f;
    }
    if (src >= 0) { p.order[lane] = src; p.lab[lane] = (int)p.labels[src]; }
    if (lane == 0) *p.nvalid = nv;
  }
  const int n0 = blockIdx.x * 256, v0 = n0 + wave * 32;
  // W and h by LDS-DMA, 64 columns at a time, three slots (straight from memory into MFMA operands, 64 B of a row per load, W came at 2.5 - 3.5 TB/s): wave w
  // fills and reads rows [32 w, 32 w + 32) of W in four pieces of 8 rows x 128 B, and fills rows [8 w, 8 w + 8) of h.  Chunk c of row r at c ^ ((r >> 1) & 7).
  const ns_u4v rsrc = ll_rsrc((const E*)p.w + (int64_t)n0 * p.ldw), rsrc_h = ll_rsrc(p.h);
  const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)smem;
  uint32_t off[4], off_h;
  int col[4], col_h;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 32 * wave + 8 * j + (lane >> 3);
    col[j] = ((lane & 7) ^ ((r >> 1) & 7)) * 8;
    off[j] = n0 + r < p.V ? (uint32_t)(r * (int)p.ldw + col[j]) * 2u : OUT;
  }
  {
    const int r = 8 * wave + (lane >> 3), at = __shfl(src, r, 64);
    col_h = ((lane & 7) ^ ((r >> 1) & 7)) * 8;
    off_h = at >= 0 ? (uint32_t)(at * (int)p.ldh + col_h) * 2u : OUT;
  }
  const int chunks = (p.d + 63) / 64;
  auto stage = [&](int c) __attribute__((always_inline)) {
    const bool in = c < chunks;
    const uint32_t dst = lds_base + (c % 3) * FW_BYTES + wave * 4096;
#pragma unroll
    for (int j = 0; j < 4; ++j) ll_dma16(rsrc, in && c * 64 + col[j] < p.d ? off[j] : OUT, in ? c * 128 : 0, dst + j * 1024);
    ll_dma16(rsrc_h, in && c * 64 + col_h < p.d ? off_h : OUT, in ? c * 128 : 0, lds_base + 3 * FW_BYTES + (c % 3) * FH_BYTES + wave * 1024);
  };
  f32x4 acc[2][MT];
#pragma unroll
  for (int f = 0; f < 2; ++f)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[f][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  stage(0);
  stage(1);
  for (int c = 0; c < chunks; ++c) {
    stage(c + 2);
    asm volatile("s_waitcnt vmcnt(10)" ::: "memory");          // chunk c has landed (this wave's pieces; the barrier covers the others)
    LL_BARRIER();
    const char* const ws = smem + (c % 3) * FW_BYTES + (wave * 32 + l15) * 128;
    const char* const hs = smem + 3 * FW_BYTES + (c % 3) * FH_BYTES + l15 * 128;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int at = ((4 * ks + lg) ^ (l15 >> 1)) << 4;        // (16 rows further: the same permutation)
      v8 a[2];
#pragma unroll
      for (int f = 0; f < 2; ++f) a[f] = *(const v8*)(ws + f * 2048 + at);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const v8 b = *(const v8*)(hs + m * 2048 + at);
#pragma unroll
        for (int f = 0; f < 2; ++f) acc[f][m] = T::mma(a[f], b, acc[f][m]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    LL_BARRIER();                                              // everyone has read this chunk before its slot is filled again
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  // a lane holds 4 neighbouring tokens of 16 MT rows, twice
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = m * 16 + l15;
    float mx = -INFINITY;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (r < nv) *(f32x4*)(p.z + (int64_t)r * p.ldz + v0 + f * 16 + 4 * lg) = acc[f][m];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (v0 + f * 16 + 4 * lg + e >= p.V) acc[f][m][e] = -INFINITY;
        mx = fmaxf(mx, acc[f][m][e]);
      }
    }
    mx = ll_max4(mx);
    const float e1 = mx == -INFINITY ? 0.f : ll_ref(mx, p.c1), e2 = mx == -INFINITY ? 0.f : ll_ref(mx, p.c2);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[f][m][e], p.c1, -e1));
        if (DUAL) s2 += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[f][m][e], p.c2, -e2));
      }
    s1 = ll_sum4(s1);
    if (DUAL) s2 = ll_sum4(s2);
    if (lg == 0) { sm[0][wave][r] = mx; sm[1][wave][r] = s1; if (DUAL) sm[2][wave][r] = s2; }
  }
  __syncthreads();
  if (tid < 16 * MT) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < 8; ++w) mx = fmaxf(mx, sm[0][w][tid]);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float m = sm[0][w][tid];
      s1 += sm[1][w][tid] * (m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(m, p.c1) - ll_ref(mx, p.c1)));      // (a NaN stays one)
      if (DUAL) s2 += sm[2][w][tid] * (m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ll_ref(m, p.c2) - ll_ref(mx, p.c2)));
    }
    const int64_t o = (int64_t)blockIdx.x * p.R + tid;
    p.pm[o] = mx;
    p.p1[o] = s1;
    if (DUAL) p.p2[o] = s2;
  }
}

constexpr int FG_LD = 256 * 2 + 16;          // bytes per staged row of dz
template <int MT> constexpr int few_lds() { return 3 * FW_BYTES + 3 * FH_BYTES + 16 * MT * FG_LD; }

// grid (tiles_n, column groups).  K of dW is the rows, padded to 32 with zeros.
template <class T, int MT, bool DUAL>
__global__ __launch_bounds__(512) void ll_few_grad_kernel(const FewArgs p) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  typedef typename T::e E;
  typedef typename T::v8 v8;
  typedef E e4 __attribute__((ext_vector_type(4)));
  char* const hs = smem + 3 * FW_BYTES;
  char* const gs_ = hs + 3 * FH_BYTES;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * 256;
  const int chunks = (p.d + 63) / 64, per = (chunks + gridDim.y - 1) / gridDim.y;
  const int c_begin = blockIdx.y * per, c_end = min(chunks, c_begin + per);
  int src;
  const int nv = few_rows(p.labels, p.rows, p.V, lane, src);
  // Few enough rows with a label leave half of dz's rows free: row r + HALF then holds what row r's rounding lost, dh's two rows are added at the end and h's row
  // stands there twice for dW.  The label's cell is most of such a row's dz, and its one rounding would be a factor on the whole gradient: with many
  // rows these factors average out, with one fp16 row dh was off by 3.1e-4 where its own rounding is 2.1e-4.
  // Where the rows fill them (33 to 64 labels), the largest of a row's cells among these tokens counts by itself: what its rounding lost goes into the row's dh and the
  // token's dW in fp32, from W's and h's rows in LDS (48 rows, d = 512: 1.2 - 1.5 -> 1.0 times the result's own rounding).  Per row: |cell| above, its residue's upper 24
  // bits and the token below.
  constexpr int HALF = 8 * MT;
  const bool twice = nv <= HALF;
  __shared__ unsigned long long big[64];
  if (tid < 64) big[tid] = 0;
  // Chunks of 64 columns by LDS-DMA, three slots: of W (for dh) wave w fills rows [32 w, 32 w + 32) in four pieces of 8 rows x 128 B, of h (for dW) rows
  // [8 w, 8 w + 8) in one, packed rows of h by their original place.  The 32-B windows of row r are permuted by f(r) = bit 1 | bit 3 << 1, so that the eight
  // row segments of half a transposed read lie in different banks (even and odd rows already do).
  const ns_u4v rsrc = ll_rsrc((const E*)p.w + (int64_t)n0 * p.ldw), rsrc_h = ll_rsrc(p.h);
  const uint32_t lds_base = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)smem;
  uint32_t off[4], off_h;
  int col[4], col_h;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = 32 * wave + 8 * j + (lane >> 3), f = ((r >> 1) & 1) | (((r >> 3) & 1) << 1);
    col[j] = ((lane & 7) ^ (f << 1)) * 8;
    off[j] = n0 + r < p.V ? (uint32_t)(r * (int)p.ldw + col[j]) * 2u : OUT;
  }
  {
    const int r = 8 * wave + (lane >> 3), f = ((r >> 1) & 1) | (((r >> 3) & 1) << 1), at = __shfl(src, twice && r >= HALF ? r - HALF : r, 64);
    col_h = ((lane & 7) ^ (f << 1)) * 8;
    off_h = at >= 0 ? (uint32_t)(at * (int)p.ldh + col_h) * 2u : OUT;
  }
  auto stage = [&](int c) __attribute__((always_inline)) {
    const bool in = c < c_end;
    if (p.dh) {
      const uint32_t dst = lds_base + (c % 3) * FW_BYTES + wave * 4096;
#pragma unroll
      for (int j = 0; j < 4; ++j) ll_dma16(rsrc, in && c * 64 + col[j] < p.d ? off[j] : OUT, in ? c * 128 : 0, dst + j * 1024);
    }
    if (p.dw) ll_dma16(rsrc_h, in && c * 64 + col_h < p.d ? off_h : OUT, in ? c * 128 : 0, lds_base + 3 * FW_BYTES + (c % 3) * FH_BYTES + wave * 1024);
  };
  stage(c_begin);
  stage(c_begin + 1);
  // dz of these 256 tokens
  for (int x = tid; x < 16 * MT * 64; x += 512) {
    const int r = x >> 6, c = (x & 63) * 4;
    if (twice && r >= HALF) break;
    float g[4] = {0.f, 0.f, 0.f, 0.f};
    if (r < nv) {
      const f32x4 z = *(const f32x4*)(p.z + (int64_t)r * p.ldz + n0 + c);
      const float la = p.La[r], lb = DUAL ? p.Lb[r] : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        g[e] = __builtin_amdgcn_exp2f(z[e] * p.c1 - la);
        if (DUAL) g[e] += __builtin_amdgcn_exp2f(z[e] * p.c2 - lb);
        if (n0 + c + e >= p.V) g[e] = 0.f;
      }
    }
    *(ushort4v*)(gs_ + r * FG_LD + c * 2) = cvt4<E>(g[0], g[1], g[2], g[3]);
    if (twice)
      *(ushort4v*)(gs_ + (r + HALF) * FG_LD + c * 2) = cvt4<E>(g[0] - (float)(E)g[0], g[1] - (float)(E)g[1], g[2] - (float)(E)g[2], g[3] - (float)(E)g[3]);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  LL_BARRIER();
  // its sparse cells: entries 0 .. k - 1 the list, k the label; an entry whose token an earlier one names is written by that one
  for (int x = tid; x < nv * (p.k + 1); x += 512) {
    const int r = x / (p.k + 1), e = x - r * (p.k + 1);
    const int lab = p.lab[r], row = p.order[r];
    const int t = e == p.k ? lab : p.top_idx[row * p.ld_top + e];
    if (t < n0 || t >= n0 + 256 || t >= p.V) continue;
    float soft = 0.f;
    bool first = true;
    const RowK kk = ll_row_k(p.rk + r * LL_RK);
    const float z = p.z[(int64_t)r * p.ldz + t];
#pragma unroll 8
    for (int o = 0; o < p.k; ++o)
      if (p.top_idx[row * p.ld_top + o] == t) { soft += p.pk[(int64_t)r * p.k + o]; first = first && o >= e; }
    if (!first) continue;
    const float v = ll_sparse_cell(kk, z, p.c1, p.c2, p.w1s, p.w2s, soft, t == __float_as_int(kk.hi[RK_TOKEN - 4]), t == lab);
    *(E*)(gs_ + r * FG_LD + (t - n0) * 2) = (E)v;
    const float lost = v - (float)(E)v;
    if (twice) *(E*)(gs_ + (r + HALF) * FG_LD + (t - n0) * 2) = (E)lost;
    else if (p.k == 0 || fabsf(v) * 16.f >= p.w1s * kk.hi[RK_REST1 - 4] + p.w2s * kk.hi[RK_REST2 - 4])      // (of a list the small ones stay: 64 rows, 64 entries: 125 -> 117 us)
      atomicMax(&big[r], (unsigned long long)(__float_as_uint(v) & 0x7FFFFFFFu) << 32 | (__float_as_uint(lost) & 0xFFFFFF00u) | (unsigned)(t - n0));
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  LL_BARRIER();
  auto tr8 = [&](const char* at, int four_rows) __attribute__((always_inline)) {      // 8 k-rows of 16 columns, transposed
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + four_rows));
    const short8v r = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(v8, r);
  };
  const int q = l15 >> 2, pp = l15 & 3;
  const float gs = (p.loss_scale ? *p.loss_scale : 1.f) / (float)max(nv, 1) * p.unscale;
  // dW: this wave's 32 tokens as the MFMA's columns (dz transposed), the rows as K (16 rows: the upper half of a K step is zero)
  constexpr int KS = MT < 2 ? 1 : MT / 2;
  v8 gt[2][KS];
  if (p.dw) {
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int rr = MT == 1 ? 8 * (lg & 1) + q : ks * 32 + 8 * lg + q;
        const v8 v = tr8(gs_ + rr * FG_LD + (wave * 32 + f * 16 + 4 * pp) * 2, 4 * FG_LD);
        gt[f][ks] = MT == 1 && lg >= 2 ? v8{} : v;
      }
  }
  // this lane's row of dh's blocks, and which rows' cells lie in this wave's 32 tokens
  constexpr int NB = MT < 2 ? 1 : MT / 2;
  int row_tok[NB];
  float row_lost[NB];
  uint64_t mine = 0;
  unsigned long long at_lane = 0;
  if (!twice) {
    at_lane = big[lane];
    mine = __ballot(at_lane != 0 && (int)((unsigned)at_lane & 255) >> 5 == wave);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const unsigned long long b = big[((n * 8 + wave) >> 2) * 16 + l15 & 63];
      row_tok[n] = b ? (int)((unsigned)b & 255) : -1;
      row_lost[n] = __uint_as_float((unsigned)b & 0xFFFFFF00u);
    }
  }
  // how many stores a wave issues behind a chunk's pieces in a full chunk (fewer in a ragged one: there the waits count none)
  const bool full_v = n0 + 256 <= p.V;
  for (int c = c_begin; c < c_end; ++c) {
    stage(c + 2);
    // chunk c has landed when, behind it, only chunk c + 1, the stores of step c - 1 and chunk c + 2 may be in flight (this wave's; the barrier covers the others)
    const bool counted = full_v && c > c_begin && !p.f32;     // (step c - 1 is a full chunk: only the last may be ragged)
    constexpr int SH = MT / 2;                                // stores of dh per wave and step (16 rows: half of the waves have one, not counted)
    if (p.dh && p.dw) {
      if (counted) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(14 + SH) : "memory");      // 5 + 4 + SH + 5
      else asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    } else if (p.dh) {
      if (c > c_begin) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(8 + SH) : "memory");   // 4 + SH + 4
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      if (counted) asm volatile("s_waitcnt vmcnt(6)" ::: "memory");                    // 1 + 4 + 1
      else asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    LL_BARRIER();
    f32x4 dha[MT < 2 ? 1 : MT / 2];
    if (p.dh) {
      // output block `id` = (16 rows, 16 of the chunk's 64 columns), K = the 256 tokens
      const char* const ws = smem + (c % 3) * FW_BYTES;
#pragma unroll
      for (int n = 0; n < (MT < 2 ? 1 : MT / 2); ++n) {
        const int id = n * 8 + wave;
        dha[n] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (id < 4 * MT) {
          const int mt = id >> 2, ct = id & 3;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const int r = ks * 32 + 8 * lg + q, f = ((r >> 1) & 1) | (((r >> 3) & 1) << 1);      // (four rows further: the same f)
            const v8 wt = tr8(ws + r * 128 + ((ct ^ f) << 5) + pp * 8, 512);
            const v8 g = *(const v8*)(gs_ + (mt * 16 + l15) * FG_LD + (ks * 32 + 8 * lg) * 2);
            dha[n] = T::mma(wt, g, dha[n]);
          }
          if (!twice && row_tok[n] >= 0) {
            const int r = row_tok[n], f = ((r >> 1) & 1) | (((r >> 3) & 1) << 1);
            const e4 l = *(const e4*)(ws + r * 128 + ((ct ^ f) << 5) + lg * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) dha[n][e] = __builtin_fmaf(row_lost[n], (float)l[e], dha[n][e]);
          }
        }
      }
    }
    f32x4 da[4][2];
    if (p.dw) {
      const char* const hc = hs + (c % 3) * FH_BYTES;
#pragma unroll
      for (int ct = 0; ct < 4; ++ct) {
        v8 ht[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int r = ks * 32 + 8 * lg + q, f = ((r >> 1) & 1) | (((r >> 3) & 1) << 1);
          ht[ks] = tr8(hc + r * 128 + ((ct ^ f) << 5) + pp * 8, 512);
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) a = T::mma(ht[ks], gt[f][ks], a);
          da[ct][f] = a * gs;
        }
      }
      for (uint64_t m = mine; m; m &= m - 1) {
        const int r = __builtin_ctzll(m), low = __builtin_amdgcn_readlane((int)(unsigned)at_lane, r), rf = ((r >> 1) & 1) | (((r >> 3) & 1) << 1);
        const float lost = __uint_as_float((unsigned)low & 0xFFFFFF00u) * gs;
        if (l15 != (low & 15)) continue;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          const e4 x = *(const e4*)(hc + r * 128 + ((ct ^ rf) << 5) + lg * 8);
#pragma unroll
          for (int f = 0; f < 2; ++f)
            if ((low >> 4 & 1) == f) {
#pragma unroll
              for (int e = 0; e < 4; ++e) da[ct][f][e] = __builtin_fmaf(lost, (float)x[e], da[ct][f][e]);
            }
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    LL_BARRIER();                                              // everyone has read this chunk before its slot is filled again
    if (p.dw) {
      if (p.f32) {
#pragma unroll
        for (int ct = 0; ct < 4; ++ct)
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const int v = n0 + wave * 32 + f * 16 + l15, cc = c * 64 + ct * 16 + 4 * lg;
            if (v >= p.V || cc >= p.d) continue;
            f32x4* const at = (f32x4*)((float*)p.dw + (int64_t)v * p.lddw + cc);
            *at = p.add ? *at + da[ct][f] : da[ct][f];
          }
      } else {
        // two column blocks of 16: the lanes of odd 16-lane rows give their 4 columns of the first for the even rows' 4 of the second, so that a lane holds 8
        // neighbouring columns (16 B) and four lanes 64 B of a row of W
#pragma unroll
        for (int cp = 0; cp < 2; ++cp)
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            typedef unsigned u2 __attribute__((ext_vector_type(2)));
            const f32x4 x = da[2 * cp][f], y = da[2 * cp + 1][f];
            const u2 xa = __builtin_bit_cast(u2, cvt4<E>(x[0], x[1], x[2], x[3])), ya = __builtin_bit_cast(u2, cvt4<E>(y[0], y[1], y[2], y[3]));
            const u2 r0 = __builtin_amdgcn_permlane16_swap(xa[0], ya[0], false, false), r1 = __builtin_amdgcn_permlane16_swap(xa[1], ya[1], false, false);
            const int v = n0 + wave * 32 + f * 16 + l15, cc = c * 64 + (2 * cp + (lg & 1)) * 16 + (lg >> 1) * 8;
            if (v < p.V && cc < p.d) *(uint4*)((E*)p.dw + (int64_t)v * p.lddw + cc) = make_uint4(r0[0], r1[0], r0[1], r1[1]);
          }
      }
    }
    if (p.dh) {
#pragma unroll
      for (int n = 0; n < (MT < 2 ? 1 : MT / 2); ++n) {
        const int id = n * 8 + wave, mt = id >> 2, ct = id & 3, cc = c * 64 + ct * 16 + 4 * lg;
        if (id < 4 * MT && cc < p.d) *(f32x4*)(p.slab + ((int64_t)blockIdx.x * 16 * MT + mt * 16 + l15) * p.d + cc) = dha[n];
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ------------------------------------------------------------------------------------------------ host
struct Plan {
  int few;                                    // 0, or MT of the few-row path
  int keep, ref, R, Rc, dp, dt, tiles_n, piece_tiles, pieces, pairs;      // keep: LL_KEEP, in chunks of Rc rows (else Rc = R, in pieces of the vocabulary)
  size_t splits_at, order, inv, lab, xtok, xz, hp, hT, zk, pk, pm, p1, p2, strip, La, Lb, rk, eref, efin, F, big, ploss, G, slab, total;
};

bool dual_of(const ns_linear_ce_desc* d) { return d->k > 0 && d->alpha > 0.f && d->alpha < 1.f && d->temperature != 1.f; }

Plan plan_of(const ns_linear_ce_desc* d) {
  Plan p = {};
  const int parts = d->dh || d->dw ? 2 : 1;       // (a cell in two parts takes two rows of dz, ll_few_grad: 12 rows 39 -> 42 us, 30 rows 44 -> 52)
  p.few = d->rows > LL_FEW_ROWS ? 0 : d->rows * parts <= 16 ? 1 : d->rows * parts <= 32 ? 2 : 4;
  p.R = (d->rows > 0 ? d->rows + BM - 1 : BM) / BM * BM;
  p.dp = (d->d + BK - 1) / BK * BK;
  p.dt = (d->d + BM - 1) / BM * BM;
  p.tiles_n = (d->vocab + BN - 1) / BN;
  const bool grad = d->dh || d->dw;
  // Either whole rows of 16-bit exponentials in chunks of rows, no logit formed twice: one softmax, or two at 1 <= T <= 2, and dW not spread over chunks; or dz of one piece of the
  // vocabulary at a time for all rows.  A k-range of the head, and for dW all rows of dz, are addressed with 32-bit byte offsets (LL_WHOLE_BYTES < 2^31).
  const int64_t ldw = d->ldw > d->d ? d->ldw : d->d;
  const int64_t by_ld = ((int64_t)0x7FF00000 / 2 / ldw) / BN;
  const int64_t rows_fit = (int64_t)((d->dw ? LL_WHOLE_BYTES : LL_PIECE_BYTES) / ((size_t)p.tiles_n * BN * 2)) / BM * BM;
  p.keep = grad && (!dual_of(d) || d->temperature <= 2.f && d->temperature >= 1.f) && rows_fit >= BM && p.tiles_n <= by_ld && (p.R <= rows_fit || !d->dw);
  p.ref = p.keep && !p.few && !dual_of(d) && (d->k == 0 ? d->dtype == NS_BF16 || !d->dw : d->dtype == NS_BF16 && !d->dw);
  p.Rc = p.R;
  if (p.keep) {
    if (p.R > rows_fit) {
      const int n = (int)((p.R + rows_fit - 1) / rows_fit);
      p.Rc = ((p.R / BM + n - 1) / n) * BM;
    }
    p.pieces = 1;
    p.piece_tiles = p.tiles_n;
  } else {
    int64_t most = (int64_t)(LL_PIECE_BYTES / ((size_t)p.R * BN * 2));
    if (most > by_ld) most = by_ld;
    if (most < 1) most = 1;
    p.pieces = (int)((p.tiles_n + most - 1) / most);
    p.piece_tiles = (p.tiles_n + p.pieces - 1) / p.pieces;
    p.pieces = (p.tiles_n + p.piece_tiles - 1) / p.piece_tiles;
  }
  // dh's slabs: one 256 x 256 fp32 tile per (output tile, split of the piece's vocabulary)
  const int tiles = (p.Rc / BM) * ((d->d + BN - 1) / BN), kt = p.piece_tiles * (BN / BK);
  p.pairs = tiles;                                 // (fewer live tiles may be split more ways: at most LL_PAIRS pairs, or kt / 8 a tile)
  if (p.pairs < LL_PAIRS) p.pairs = (int64_t)tiles * (kt / 8) < LL_PAIRS ? (tiles * (kt / 8) > tiles ? tiles * (kt / 8) : tiles) : LL_PAIRS;
  if (p.few) p.R = p.Rc = LL_FEW_ROWS;
  size_t at = 0;
  auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) / 256 * 256; return o; };
  p.splits_at = take(4);
  p.order = take((size_t)d->rows * 4);
  p.inv = take((size_t)d->rows * 4);
  p.lab = take((size_t)d->rows * 4);
  p.xtok = p.few ? 0 : take((size_t)p.R * 4);
  p.hp = p.few ? 0 : take((size_t)p.R * p.dp * 2);
  p.hT = d->dw && !p.few ? take((size_t)p.dt * p.R * 2) : 0;
  p.zk = take(p.few ? (size_t)16 * p.few * p.tiles_n * BN * 4 : (size_t)p.R * (d->k + 1) * 4);       // (few rows: all logits)
  p.xz = p.few ? 0 : d->k == 0 ? p.zk : take((size_t)p.R * 4);
  p.pk = take((size_t)p.R * d->k * 4);
  p.pm = take((size_t)p.tiles_n * p.Rc * 4);
  p.p1 = take((size_t)p.tiles_n * p.Rc * 4);
  p.p2 = dual_of(d) ? take((size_t)p.tiles_n * p.Rc * 4) : 0;
  p.strip = p.keep && !p.few ? take((size_t)p.tiles_n * 4 * p.Rc * 4) : 0;
  p.La = take((size_t)p.Rc * 4);
  p.Lb = take((size_t)p.Rc * 4);
  p.rk = take((size_t)p.Rc * LL_RK * 4);
  p.eref = p.ref ? take((size_t)p.R * 4) : 0;
  p.efin = p.ref ? take((size_t)p.Rc * 4) : 0;
  p.F = p.ref ? take((size_t)p.Rc * 4) : 0;
  p.big = grad && !p.few && !(p.ref && d->k == 0) ? take((size_t)p.R * 16) : 0;
  p.ploss = take((size_t)p.R * 4);
  p.G = grad && !p.few ? take((size_t)p.Rc * p.piece_tiles * BN * 2) : 0;
  p.slab = d->dh ? take(p.few ? (size_t)p.tiles_n * 16 * p.few * d->d * 4 : (size_t)p.pairs * BM * BN * 4) : 0;
  p.total = at;
  return p;
}

// groups of slabs that ll_dh_out_kernel adds side by side
int dh_groups(const Plan& p) { return p.few ? (p.tiles_n >= 64 ? 16 : p.tiles_n >= 16 ? 4 : 1) : p.Rc <= 512 ? 16 : 1; }

bool ll_sizes_ok(const ns_linear_ce_desc* d) {
  return d->rows >= 0 && d->rows <= (1 << 21) && d->vocab > 0 && d->vocab <= (1 << 28) && d->d > 0 && d->d % 8 == 0 && d->d <= (1 << 16) && d->k >= 0 && d->k <= LL_MAX_K;
}

template <class T, int MT>
int few_launch(const ns_linear_ce_desc* d, const Plan& p, const FewArgs& f, const RowArgs& r, bool dual, hipStream_t st) {
  typedef typename T::e E;
  static ns_dev_once once;
  if (!ns_dyn_lds_once(once, {(const void*)ll_few_grad_kernel<T, MT, false>, (const void*)ll_few_grad_kernel<T, MT, true>, (const void*)ll_few_logits_kernel<T, MT, false>,
                              (const void*)ll_few_logits_kernel<T, MT, true>}, few_lds<MT>() > FL_LDS ? few_lds<MT>() : FL_LDS, "ns_linear_cross_entropy"))
    return NS_ERR_HIP;
  if (dual) hipLaunchKernelGGL((ll_few_logits_kernel<T, MT, true>), dim3(f.tiles_n), dim3(512), FL_LDS, st, f);
  else hipLaunchKernelGGL((ll_few_logits_kernel<T, MT, false>), dim3(f.tiles_n), dim3(512), FL_LDS, st, f);
  hipLaunchKernelGGL(ll_rows_kernel<1024>, dim3(1), dim3(1024), 0, st, r);
  if (d->dh || d->dw) {
    // a workgroup per CU: where the vocabulary is small, its column chunks are dealt to several
    const int chunks = (d->d + 63) / 64;
    int gy = 256 / f.tiles_n;
    if (gy < 1) gy = 1;
    if (gy > chunks) gy = chunks;
    gy = (chunks + (chunks + gy - 1) / gy - 1) / ((chunks + gy - 1) / gy);
    if (dual) hipLaunchKernelGGL((ll_few_grad_kernel<T, MT, true>), dim3(f.tiles_n, gy), dim3(512), few_lds<MT>(), st, f);
    else hipLaunchKernelGGL((ll_few_grad_kernel<T, MT, false>), dim3(f.tiles_n, gy), dim3(512), few_lds<MT>(), st, f);
    if (d->dh) launch_dh_out<E>(f.slab, dh_groups(p), f.tiles_n, nullptr, 16 * MT, 0, LL_FEW_ROWS, d->d, d->rows, f.inv, d->nvalid_dev, d->loss_scale_dev, f.unscale, (E*)d->dh, d->lddh, nullptr, nullptr, nullptr, nullptr, 0, nullptr, nullptr, nullptr, nullptr, st);
  }
  NS_CHECK_LAUNCH("ns_linear_cross_entropy");
  return NS_OK;
}

template <class T>
int ll_launch(const ns_linear_ce_desc* d, const Plan& p, hipStream_t st) {
  typedef typename T::e E;
  char* const ws = (char*)d->workspace;
  int *order = (int*)(ws + p.order), *inv = (int*)(ws + p.inv), *lab = (int*)(ws + p.lab);
  int* const splits = (int*)(ws + p.splits_at);
  float *zk = (float*)(ws + p.zk), *pk = (float*)(ws + p.pk), *La = (float*)(ws + p.La), *Lb = (float*)(ws + p.Lb), *ploss = (float*)(ws + p.ploss), *rk = (float*)(ws + p.rk), *xz = (float*)(ws + p.xz);
  int* const xtok = (int*)(ws + p.xtok);
  float *const eref = p.ref ? (float*)(ws + p.eref) : nullptr, *const efin = p.ref ? (float*)(ws + p.efin) : nullptr, *const F = p.ref ? (float*)(ws + p.F) : nullptr;
  const bool apart = p.ref && d->k == 0;                           // dz without the labels' cells: dh's last step adds their rows of W, dW's their rows of h
  int* const big_tok = p.big ? (int*)(ws + p.big) : nullptr;
  float* const big_res = p.big ? (float*)(ws + p.big) + 2 * (size_t)p.R : nullptr;
  const bool dual = dual_of(d), soft_only = d->k > 0 && d->alpha == 1.f, grad = d->dh || d->dw;
  const float alpha = d->k > 0 ? d->alpha : 0.f, T_ = d->k > 0 ? d->temperature : 1.f;
  const float w1 = 1.f - alpha, w2 = alpha * T_;
  // fp16 cells of dz: |w1 + w2| <= 2^x  =>  2^s with s = 15 - x keeps them below 2^15
  int s = 0;
  if (d->dtype == NS_F16) {
    s = 15;
    for (float b = 1.f; b < w1 + w2; b *= 2.f) --s;
  }
  const float up = ldexpf(1.f, s);
  static ns_dev_once once;
  if (!ns_dyn_lds_once(once, {(const void*)ll_logits_kernel<T, LL_STATS, false, false>, (const void*)ll_logits_kernel<T, LL_STATS, true, false>,
                              (const void*)ll_logits_kernel<T, LL_KEEP, true, false>, (const void*)ll_logits_kernel<T, LL_GRAD, false, true>,
                              (const void*)ll_logits_kernel<T, LL_KEEP, false, false, false, true>, (const void*)ll_logits_kernel<T, LL_KEEP, false, false>, (const void*)ll_logits_kernel<T, LL_STATS, true, false, true>, (const void*)ll_logits_kernel<T, LL_KEEP, true, false, true>,
                              (const void*)ll_logits_kernel<T, LL_GRAD, false, false>, (const void*)ll_logits_kernel<T, LL_GRAD, true, false>,
                              (const void*)ll_dh_kernel<T>, (const void*)ll_dw_kernel<T>}, LL_LOGITS_LDS > LL_LDS ? LL_LOGITS_LDS : LL_LDS, "ns_linear_cross_entropy"))
    return NS_ERR_HIP;
  const float c1 = soft_only ? LOG2E / T_ : LOG2E, c2 = LOG2E / T_;
  RowArgs r = {};
  r.pm = (float*)(ws + p.pm); r.p1 = (float*)(ws + p.p1); r.p2 = (float*)(ws + p.p2); r.tiles_n = p.tiles_n; r.R = p.R; r.k = d->k; r.V = d->vocab;
  r.c1 = c1; r.c2 = c2; r.invT = 1.f / T_; r.w1 = w1; r.w2 = w2; r.kd = alpha * T_ * T_;
  r.lw1 = (d->k > 0 && !dual) ? (float)s : log2f(w1) + (float)s;
  r.lw2 = log2f(w2) + (float)s;
  r.dual = dual; r.soft_only = soft_only; r.nvalid = d->nvalid_dev; r.order = order; r.lab = lab; r.zk = zk; r.top_vals = d->top_vals; r.top_idx = d->top_idx;
  r.eref = eref; r.efin = efin; r.F = F; r.head = T::HEAD; r.low = log2f((float)d->vocab) + T::LOW; r.shift = (float)s; r.cl = apart ? Lb : nullptr; r.f16 = d->dtype == NS_F16; r.big_tok = d->k == 0 ? big_tok : nullptr; r.big_res = big_res;      // (one softmax: Lb is free)
  r.xtok = xtok; r.xz = xz; r.rk = grad ? rk : nullptr; r.up = up;
  r.ld_top = d->ld_top; r.La = La; r.Lb = dual ? Lb : nullptr; r.pk = pk; r.row_loss = d->row_loss; r.packed_loss = ploss; r.loss = d->loss_dev;
  if (p.few) {
    FewArgs f = {};
    f.h = d->h; f.ldh = d->ldh; f.w = d->w; f.ldw = d->ldw; f.labels = d->labels; f.rows = d->rows; f.d = d->d; f.V = d->vocab; f.tiles_n = p.tiles_n;
    f.c1 = c1; f.c2 = c2; f.z = zk; f.ldz = (int64_t)p.tiles_n * BN; f.pm = (float*)(ws + p.pm); f.p1 = (float*)(ws + p.p1); f.p2 = (float*)(ws + p.p2); f.R = p.R;
    f.order = order; f.inv = inv; f.lab = lab; f.nvalid = d->nvalid_dev; f.row_loss = d->row_loss;
    f.La = La; f.Lb = dual ? Lb : nullptr; f.pk = pk; f.rk = rk; f.top_idx = d->top_idx; f.ld_top = d->ld_top; f.k = d->k; f.w1s = w1 * up; f.w2s = w2 * up; f.unscale = 1.f / up;
    f.loss_scale = d->loss_scale_dev; f.slab = (float*)(ws + p.slab); f.dw = d->dw; f.lddw = d->lddw; f.f32 = d->dw_f32; f.add = d->dw_add; f.dh = d->dh != nullptr;
    r.z = zk; r.ldz = f.ldz;
    return p.few == 1 ? few_launch<T, 1>(d, p, f, r, dual, st) : p.few == 2 ? few_launch<T, 2>(d, p, f, r, dual, st) : few_launch<T, 4>(d, p, f, r, dual, st);
  }
  hipLaunchKernelGGL(ll_compact_kernel, dim3(1), dim3(1024), 0, st, d->labels, d->rows, d->vocab, order, inv, lab, d->row_loss, d->nvalid_dev);
  hipLaunchKernelGGL(ll_pack_kernel<T>, dim3(p.R / 4), dim3(256), 0, st, d->h, d->ldh, d->w, d->ldw, d->d, p.dp, order, lab, d->k, d->nvalid_dev, (void*)(ws + p.hp), zk, c1, eref, xtok);
  if (d->k > 0)
    hipLaunchKernelGGL(ll_gather_kernel<T>, dim3(p.R), dim3(256), 0, st, (const void*)(ws + p.hp), p.dp, d->w, d->ldw, d->d, d->vocab, order, lab, d->top_idx, d->ld_top, d->k,
                       d->nvalid_dev, zk, c1, eref, xtok, xz);
  auto transpose = [&] {
    hipLaunchKernelGGL(ll_transpose_kernel, dim3(p.R / 64, p.dp / 64), dim3(256), 0, st, (const uint16_t*)(ws + p.hp), p.dp, d->nvalid_dev, (uint16_t*)(ws + p.hT), p.R, F);
  };
  if (d->dw && !p.ref) transpose();
  LogitsArgs a = {};
  a.hp = ws + p.hp; a.w = d->w; a.ldw = d->ldw; a.dp = p.dp; a.d = d->d; a.V = d->vocab; a.col0 = 0; a.tiles_n = p.tiles_n; a.R = p.Rc; a.nvalid = d->nvalid_dev;
  a.c1 = c1; a.c2 = c2; a.T = T_;
  a.pm = (float*)(ws + p.pm); a.p1 = (float*)(ws + p.p1); a.p2 = (float*)(ws + p.p2);
  a.La = La; a.Lb = Lb; a.G = ws + p.G; a.ldg = p.piece_tiles * BN; a.lab = lab; a.rk = rk;
  a.eref = eref; a.efin = efin; a.xtok = xtok;
  a.strip = (float*)(ws + p.strip); a.shift = (float)s; a.unshift = 1.f / up;
  r.R = p.Rc; r.tiles_d = (d->d + BN - 1) / BN; r.kt = p.piece_tiles * (BN / BK); r.splits = splits;
  auto grid_of = [&](int tiles_n) { const int64_t t = (int64_t)(p.Rc / BM) * tiles_n; return dim3((unsigned)(t < 256 ? t : 256)); };
  for (int row0 = 0; row0 < p.R; row0 += p.Rc) {
    a.row0 = r.row0 = row0;
    a.col0 = 0; a.tiles_n = p.tiles_n;
    const dim3 all = grid_of(p.tiles_n);
    if (p.ref) hipLaunchKernelGGL((ll_logits_kernel<T, LL_KEEP, false, false, false, true>), all, dim3(NTH), LL_LOGITS_LDS, st, a);
    else if (p.keep && dual && T_ == 2.f) hipLaunchKernelGGL((ll_logits_kernel<T, LL_KEEP, true, false, true>), all, dim3(NTH), LL_LOGITS_LDS, st, a);
    else if (dual && T_ == 2.f) hipLaunchKernelGGL((ll_logits_kernel<T, LL_STATS, true, false, true>), all, dim3(NTH), LL_LOGITS_LDS, st, a);
    else if (p.keep && dual) hipLaunchKernelGGL((ll_logits_kernel<T, LL_KEEP, true, false>), all, dim3(NTH), LL_LOGITS_LDS, st, a);
    else if (p.keep) hipLaunchKernelGGL((ll_logits_kernel<T, LL_KEEP, false, false>), all, dim3(NTH), LL_LOGITS_LDS, st, a);
    else if (dual) hipLaunchKernelGGL((ll_logits_kernel<T, LL_STATS, true, false>), all, dim3(NTH), LL_LOGITS_LDS, st, a);
    else hipLaunchKernelGGL((ll_logits_kernel<T, LL_STATS, false, false>), all, dim3(NTH), LL_LOGITS_LDS, st, a);
    hipLaunchKernelGGL(ll_rows_kernel<256>, dim3(p.Rc / 16), dim3(256), 0, st, r);
    if (!d->dh && row0 + p.Rc >= p.R) hipLaunchKernelGGL(ll_mean_kernel, dim3(1), dim3(1024), 0, st, ploss, d->nvalid_dev, d->loss_dev);
    if (!grad) continue;
    if (d->dw && p.ref) transpose();      // (with the rows' factors; dW: one chunk)
    for (int pc = 0; pc < p.pieces; ++pc) {
      a.col0 = pc * p.piece_tiles * BN;
      a.tiles_n = p.tiles_n - pc * p.piece_tiles < p.piece_tiles ? p.tiles_n - pc * p.piece_tiles : p.piece_tiles;
      const dim3 grid = grid_of(a.tiles_n);
      if (p.keep) {
        const dim3 sg((a.tiles_n + 1) / 2, p.Rc / 64);
        if (p.ref) hipLaunchKernelGGL(ll_rebase_kernel<T>, sg, dim3(256), 0, st, a);
        else if (dual) hipLaunchKernelGGL((ll_scale_kernel<T, false, true>), sg, dim3(256), 0, st, a);
        else if (d->k == 0) hipLaunchKernelGGL((ll_scale_kernel<tf16, true, false>), sg, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((ll_scale_kernel<T, false, false>), sg, dim3(256), 0, st, a);
      } else if (d->k == 0) hipLaunchKernelGGL((ll_logits_kernel<T, LL_GRAD, false, true>), grid, dim3(NTH), LL_LOGITS_LDS, st, a);
      else if (dual) hipLaunchKernelGGL((ll_logits_kernel<T, LL_GRAD, true, false>), grid, dim3(NTH), LL_LOGITS_LDS, st, a);
      else hipLaunchKernelGGL((ll_logits_kernel<T, LL_GRAD, false, false>), grid, dim3(NTH), LL_LOGITS_LDS, st, a);
      if (d->k > 0)
        hipLaunchKernelGGL(ll_cells_kernel<E>, dim3(p.Rc / 4), dim3(256), 0, st, d->nvalid_dev, row0, p.Rc, order, lab, d->top_idx, d->ld_top, d->k, zk, pk, La,
                           rk, a.c1, a.c2, w1 * up, w2 * up, a.col0, a.tiles_n * BN, d->vocab, (E*)a.G, a.ldg, efin, big_tok, big_res);
      if (d->dh) {
        DhArgs q = {};
        q.G = a.G; q.w = d->w; q.ldw = d->ldw; q.ldg = a.ldg; q.col0 = a.col0; q.cols = a.tiles_n * BN; q.V = d->vocab; q.d = d->d; q.row0 = row0; q.R = p.Rc;
        q.kt = p.piece_tiles * (BN / BK); q.splits = splits; q.add = pc > 0; q.nvalid = d->nvalid_dev; q.slab = (float*)(ws + p.slab);
        hipLaunchKernelGGL(ll_dh_kernel<T>, dim3(p.pairs), dim3(NTH), LL_LDS, st, q);
      }
      if (d->dw) {
        DwArgs q = {};
        q.hT = ws + p.hT; q.ldt = p.R; q.G = a.G; q.ldg = a.ldg; q.col0 = a.col0; q.tiles_v = a.tiles_n; q.V = d->vocab; q.d = d->d; q.row0 = row0; q.R = p.Rc;
        q.nvalid = d->nvalid_dev; q.loss_scale = d->loss_scale_dev; q.unscale = 1.f / up; q.dw = d->dw; q.lddw = d->lddw; q.f32 = d->dw_f32; q.add = d->dw_add;
        q.hp = ws + p.hp; q.dp = p.dp; q.tok = apart ? lab : big_tok; q.coef = apart ? Lb : big_res; q.per = apart ? 0 : 1;
        hipLaunchKernelGGL(ll_dw_kernel<T>, dim3(p.dt / BM * a.tiles_n), dim3(NTH), LL_LDS, st, q);
      }
    }
    if (d->dh)
      launch_dh_out<E>((const float*)(ws + p.slab), dh_groups(p), 0, splits, 0, row0, p.Rc, d->d, d->rows, inv, d->nvalid_dev, d->loss_scale_dev, 1.f / up, (E*)d->dh,
                       d->lddh, ploss, row0 + p.Rc >= p.R ? d->loss_dev : nullptr, F, (const E*)d->w, d->ldw, lab, apart ? Lb : nullptr, big_tok, big_res, st);
  }
  NS_CHECK_LAUNCH("ns_linear_cross_entropy");
  return NS_OK;
}

}  // namespace

extern "C" size_t ns_linear_ce_workspace_bytes(const ns_linear_ce_desc* d) {
  if (!d || !ll_sizes_ok(d)) return 0;
  ns_linear_ce_desc c = *d;
  if (c.alpha == 0.f) c.k = 0;       // the hard labels alone: the teacher's list is not read
  return plan_of(&c).total;
}

extern "C" int ns_linear_cross_entropy(const ns_linear_ce_desc* desc, void* stream) {
  NS_CHECK_ARG(desc, "ns_linear_cross_entropy: null descriptor");
  ns_linear_ce_desc c = *desc;
  ns_linear_ce_desc* const d = &c;
  NS_CHECK_ARG(d->w && d->loss_dev && d->nvalid_dev && (d->rows == 0 || (d->h && d->labels && d->row_loss)), "ns_linear_cross_entropy: null pointer");
  NS_CHECK_ARG(ll_sizes_ok(d), "ns_linear_cross_entropy: bad sizes rows=%d vocab=%d d=%d k=%d (d a multiple of 8, k <= %d)", d->rows, d->vocab, d->d, d->k, LL_MAX_K);
  NS_CHECK_ARG(d->dtype == NS_F16 || d->dtype == NS_BF16, "ns_linear_cross_entropy: dtype %d (NS_F16 or NS_BF16)", d->dtype);
  const int64_t lds[] = {d->ldh, d->ldw, d->dh ? d->lddh : d->ldh, d->dw ? d->lddw : d->ldw};
  for (int64_t ld : lds) NS_CHECK_ARG(ld >= d->d && ld % 8 == 0 && ld < (1 << 21), "ns_linear_cross_entropy: row stride %lld (a multiple of 8, >= d, < 2^21)", (long long)ld);
  for (const void* q : {d->h, d->w, (const void*)d->dh, (const void*)d->dw, (const void*)d->workspace})
    NS_CHECK_ARG(((size_t)q & 15) == 0, "ns_linear_cross_entropy: a tensor does not start on 16 bytes");
  NS_CHECK_ARG(d->k == 0 || (d->top_vals && d->top_idx && d->ld_top >= d->k), "ns_linear_cross_entropy: the teacher's list needs values, tokens and a row stride >= k");
  NS_CHECK_ARG(d->k == 0 || (d->temperature >= 0.05f && d->temperature <= 100.f && d->alpha >= 0.f && d->alpha <= 1.f),
               "ns_linear_cross_entropy: temperature %g in [0.05, 100], alpha %g in [0, 1]", (double)d->temperature, (double)d->alpha);
  NS_CHECK_ARG(!d->dw_add || d->dw_f32, "ns_linear_cross_entropy: only an fp32 weight gradient is added to");
  if (d->alpha == 0.f) d->k = 0;     // the hard labels alone: the teacher's list is not read
  const Plan p = plan_of(d);
  NS_CHECK_ARG(d->workspace && d->workspace_bytes >= p.total, "ns_linear_cross_entropy: workspace of %zu bytes, %zu needed", d->workspace_bytes, p.total);
  NS_CHECK_ARG((int64_t)(p.R / BM) * p.tiles_n < (1ll << 31), "ns_linear_cross_entropy: too many tiles");
  // (a launch holds less than 2^32 threads: dh is written by 16 threads per row and 64 columns, or 256)
  NS_CHECK_ARG(!d->dh || (int64_t)d->rows * ((d->d + 63) / 64) * (256 / (16 / dh_groups(p))) < (1ll << 32) - 1024, "ns_linear_cross_entropy: rows=%d of d=%d are too many for one dh", d->rows,
               d->d);
  return d->dtype == NS_F16 ? ll_launch<tf16>(d, p, (hipStream_t)stream) : ll_launch<tbf16>(d, p, (hipStream_t)stream);
}
