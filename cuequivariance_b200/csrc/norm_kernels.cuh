// Norms around an equivariant block.  Per row z and irrep block (mul channels u, dim components i, N = mul * dim values):
//
//   branch   h = x + s_u act(g_zu) y r(y)          r(t) = (sum_ui t^2 / N + eps)^-1/2
//   norm     n = w_u t r(t)                        t = h behind a branch, t = x alone
//
// With P_u = sum_i go y the derivatives need nothing else that runs over the components:
//
//   a_u = s_u act(g_u)      c = r / N sum_u a_u P_u      dy = r (a_u go - (r c) y)
//   dg_u = s_u act'(g_u) r P_u                           ds_u = sum_z act(g_u) r P_u
//
// (r c and no r^3: that leaves the range of 32 bits for blocks of 1e13 or 1e-13)
// and the same with (w, gn, h) for (a, go, y) for the norm; behind a branch its result is added to go first.
//
// What bounds them: HBM, for long blocks in 32 bits; every value is read once and written once.  A thread block is one warp with memory of
// its own, so that nothing waits for another warp.  It takes its share of rows of every slice (neighbouring irrep blocks of 1,024 values together, or
// a longer one) and brings the slice's part of a few rows into shared memory by bulk copies, a copy per lane, the next stage while it works on
// this one; 60 to 90 KB are under way per SM.  A lane owns neighbouring channels and all their components, so neither layout needs a
// transposition and sums over components need no other lane; blocks of up to 128 channels are read from shared memory into registers once.
// Results replace the operands in shared memory and leave by bulk copies.
//
// Steps, for 32,768 rows of 128x(0e+1o+2e+3o) in float32, forward + backward (HBM floor of the norm 82 + 123 us, of the gated residual
// 133 + 143, with the next norm 174 + 266): four warps on an item 120 + 158, 231 + 315, 359 + 439; a warp per slice 106 + 175, 183 + 226,
// 240 + 473; every warp on every slice 108 + 157, 156 + 178, 210 + 339; fewer warps for long blocks 100 + 146 (5.4 and 5.5 TB/s),
// 152 + 171 (5.7 and 5.5 TB/s), 214 + 310 (5.3 and 5.6 TB/s).  Short blocks, 16-bit data and codes are bound by instructions: 262,144 rows of
// 64x(0e+1o) in bfloat16 115 + 149 us (floor 72 + 82), 0.7 of the issue slots used; the gate's exponential and the sums over the warp
// are most of them.
//
// Sums, statistics and all arithmetic are in 32 bits for 16- and 32-bit data, in 64 for 64-bit data; results are rounded once.  In 16 bits
// h is rounded on its way out, so the backward pass of the norm behind a branch reads x in its place and forms h again (kAgain): as many bytes,
// and the gradients of s and w, which may have 32 bits, are not half a step of 16 bits off.  Backward in bfloat16 with h read as rounded and now:
// 32,768 rows of 128x(0e+1o+2e+3o) 208 and 217 us, 262,144 of 64x(0e+1o) 350 and 338, 32,768 of 256x(0e+1o), in loops, 246 and 279.
//
// Kept in 8 bits (Q8): codes per (row, irrep block), see code_step in common.cuh.  r stays that of the exact values; the gradients of a block
// that holds an infinity or NaN are NaN.
#pragma once
#include "common.cuh"
#include "tc_common.cuh"

namespace cueq_norm {

using cueq_tc::bar_expect_tx;
using cueq_tc::bar_init;
using cueq_tc::bar_wait;
using cueq_tc::s32;

// Params stay below 4 KB
constexpr int kMaxBlocks = CUEQ_NORM_MAX_BLOCKS;
// warps of an SM that its registers hold
__host__ __device__ constexpr int warps_per_sm(int msize) { return msize == 8 ? 8 : 16; }
constexpr int kSms = 148;
enum Mode { kBranch = 1, kNorm = 2, kBoth = 3 };

struct Blk {
  int mul, off, ch;                  // off, ch: first element of the block in a row of features, first channel
  int code, gcode, hcode;            // first byte in a row of codes: of y (or x, norm alone), of the gates, of h
  int sum;                           // first of its sums, in those of the slice
  short dim;
  unsigned char per_lane, lanes;     // neighbouring channels of a lane (0: any number, one by one), lanes of a row
};
struct Slice {
  short first, count;                // blocks
  short rps;                         // rows per stage
  short loops;                       // some block has more channels than registers hold
  int values, channels;              // of its blocks
  int sums;                          // sums per parameter: one per channel, or per channel of every row that a warp takes at a time
};
// How rows of an operand move.  kRows: a bulk copy per row; kDense: rows follow one another without a gap, one bulk copy per stage;
// kPlain: element by element, where addresses or lengths are not multiples of 16 bytes.
enum Route { kPlain, kRows, kDense };
enum Tensor { tX, tY, tG, tH, tGo, tGn, tOut, tNorm, tDx, tDy, tDg, tStats, kTensors };

struct Params {
  const void *x, *y, *g, *h, *go, *gn;
  int64_t ldx, ldy, ldg, ldh, ldgo, ldgn;
  const void *s, *w;
  void *out, *norm;                  // forward results, rows of `dim_total`
  void *dx, *dy, *dg;
  signed char* codes;
  int64_t ldc;
  void* stats;
  void* parts;                       // null: no gradients of the parameters
  int64_t rows;
  double eps;
  int* status;
  int nb, ns, dim_total, channels;   // ns: statistics per (row, block)
  int64_t deal;                      // units of rows and slices per warp; the first `deal_more` warps have one more
  int deal_more;
  int num_slices, unit, stages;      // unit: rows after which dense rows are on a 16-byte boundary again; stages: 2, or 1 where two leave room for few warps
  int pdtype, gate, mul_ir;
  signed char route[kTensors];
  Blk blk[kMaxBlocks];
  Slice slice[kMaxBlocks];
};

static_assert(sizeof(Params) <= 4000, "kernel parameters");
__host__ __device__ constexpr int pad16(int bytes) { return (bytes + 15) & ~15; }
__host__ __device__ inline int code_bytes(const Params& p, const Slice& s) {
  int n = 0;
  for (int k = s.first; k < s.first + s.count; ++k) n += pad16(p.blk[k].mul * p.blk[k].dim);
  return n;
}
__host__ __device__ inline int gate_code_bytes(const Params& p, const Slice& s) {
  int n = 0;
  for (int k = s.first; k < s.first + s.count; ++k) n += pad16(p.blk[k].mul);
  return n;
}

// Regions of a stage: byte offset, distance and length of the rows.
struct Region { int at, pitch, bytes; };
struct Stage { Region a, b, c, d, g, dg, ca, cg, ch, st; int total; };

__host__ __device__ inline Region region(bool on, int bytes, bool dense, int rps, int& at) {
  const Region r{at, dense ? bytes : pad16(bytes), bytes};
  if (on) at += pad16(r.pitch * rps);
  return r;
}
// An operand and the result that replaces it share rows: without gaps only if both are.
__host__ __device__ inline bool both_dense(const Params& p, int in, int out) { return p.route[in] == kDense && p.route[out] == kDense; }

// forward: a = x (then out, or norm alone), b = y (then norm), g = gates, ca / cg / ch = codes of y (x), gates, out
__host__ __device__ inline Stage forward_stage(const Params& p, const Slice& s, int mode, bool q8, int size) {
  Stage t{};
  const bool branch = mode & kBranch, gated = branch && p.gate != CUEQ_NORM_GATE_NONE;
  const int item = s.values * size, rps = s.rps;
  int at = 0;
  t.a = region(true, item, both_dense(p, tX, branch ? tOut : tNorm), rps, at);
  t.b = region(branch, item, mode == kBoth ? both_dense(p, tY, tNorm) : p.route[tY] == kDense, rps, at);
  t.g = region(gated, s.channels * size, p.route[tG] == kDense, rps, at);
  t.ca = region(q8, code_bytes(p, s), false, rps, at);
  t.cg = region(q8 && gated, gate_code_bytes(p, s), false, rps, at);
  t.ch = region(q8 && mode == kBoth, code_bytes(p, s), false, rps, at);
  t.total = at;
  return t;
}
// backward: a = go (then dx behind a branch with a norm, dy behind one without), b = gn (then dy, or dx for the norm alone), c = h (kAgain: x),
// d = y, g = gates, dg = their gradient (over g where that is not in codes), st = statistics
__host__ __device__ inline Stage backward_stage(const Params& p, const Slice& s, int mode, bool q8, int size, int stat_bytes) {
  Stage t{};
  const bool branch = mode & kBranch, norm = mode & kNorm, gated = branch && p.gate != CUEQ_NORM_GATE_NONE;
  const int item = s.values * size, rps = s.rps, kept = q8 ? code_bytes(p, s) : item;
  int at = 0;
  t.a = region(branch, item, mode == kBoth ? p.route[tDx] == kDense && (!p.go || p.route[tGo] == kDense) : both_dense(p, tGo, tDy), rps, at);
  t.b = region(norm, item, both_dense(p, tGn, mode == kBoth ? tDy : tDx), rps, at);
  t.c = region(norm, kept, !q8 && p.route[tH] == kDense, rps, at);
  t.d = region(branch, kept, !q8 && p.route[tY] == kDense, rps, at);
  t.g = region(gated, q8 ? gate_code_bytes(p, s) : s.channels * size, !q8 && both_dense(p, tG, tDg), rps, at);
  t.dg = t.g;
  if (q8) t.dg = region(gated, s.channels * size, p.route[tDg] == kDense, rps, at);
  t.st = region(true, s.count * stat_bytes, p.route[tStats] == kDense, rps, at);
  t.total = at;
  return t;
}
// in front of the stages: 2 barriers and the tensors' moves; then per channel, as far as the mode has them, s, w, s act(g) of the row at work (for
// the loops), and (backward) the sums of both gradients
constexpr int kMoves = 11, kMoveBytes = 40, kBars = 16 + kMoves * kMoveBytes + 8;
__host__ __device__ constexpr int pad4(int n) { return (n + 3) & ~3; }
struct Head { int s, w, a, sum_s, sum_w, total; };
__host__ __device__ inline Head head_of(const Slice& s, int mode, bool backward) {
  const int n = pad4(s.channels);
  Head h;
  h.s = 0;
  h.w = h.s + (mode & kBranch ? n : 0);
  h.a = h.w + (mode & kNorm ? n : 0);
  h.sum_s = h.a + ((mode & kBranch) && s.loops ? n : 0);
  h.sum_w = h.sum_s + (backward && (mode & kBranch) ? s.sums : 0);
  h.total = h.sum_w + (backward && (mode & kNorm) ? s.sums : 0);
  return h;
}
__host__ __device__ inline int head_bytes(int msize, const Slice& s, int mode, bool backward) { return (kBars + msize * head_of(s, mode, backward).total + 127) & ~127; }

// ---- conversions ----------------------------------------------------------------------------------------------------
template <class M> __device__ __forceinline__ M to(float v) { return (M)v; }
template <class M> __device__ __forceinline__ M to(double v) { return (M)v; }
template <class M> __device__ __forceinline__ M to(__nv_bfloat16 v) { return (M)__bfloat162float(v); }
template <class M> __device__ __forceinline__ M to(__half v) { return (M)__half2float(v); }
template <class M> __device__ __forceinline__ M to(signed char v) { return (M)(int)v; }
template <class T> __device__ __forceinline__ T from(float v);
template <class T> __device__ __forceinline__ T from(double v);
template <> __device__ __forceinline__ float from<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ double from<double>(double v) { return v; }

__device__ __forceinline__ float inverse_sqrt(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inverse_sqrt(double v) { return 1.0 / sqrt(v); }
__device__ __forceinline__ float reciprocal(float v) { return __fdividef(1.0f, v); }   // 0 from 2^126 on
__device__ __forceinline__ double reciprocal(double v) { return 1.0 / v; }
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }   // ordered as |v|, NaN above all
__device__ __forceinline__ unsigned magnitude(double) { return 0u; }                                  // 64-bit data are not kept in codes

// the fast exponential for gates of 16 bits: by CUDA's tables up to 2 + 1.173 |g| units in the last place off, so half a step of float16 is 100 times that for |g| < 8
template <class T> __device__ __forceinline__ float exponential_for(float v) { return sizeof(T) == 2 ? __expf(v) : expf(v); }
template <class T> __device__ __forceinline__ double exponential_for(double v) { return exp(v); }
template <class T, class M>
__device__ __forceinline__ void activation(int gate, M g, M& v, M& dv) {
  if (gate == CUEQ_NORM_GATE_NONE) { v = M(1); dv = M(0); return; }
  const M e = reciprocal(M(1) + exponential_for<T>(-g));
  if (gate == CUEQ_NORM_GATE_SIGMOID) { v = e; dv = e * (M(1) - e); }
  else { v = g * e; dv = e * (M(1) + g * (M(1) - e)); }
}

using cueq::code_step;
using cueq::to_code;
__device__ __forceinline__ signed char to_code(double, float) { return 0; }

// ---- one (row, irrep block) ---------------------------------------------------------------------------------------------
template <class M>
struct View {
  M *s, *w, *a, *acc_s, *acc_w;      // parameters, s act(g), sums; per channel of the block
  int mul, dim, lane, lanes, gate, gated;
  M inv_n, eps;
};

// channel u, component i: DIM 0 is a dimension known at run time only
template <int DIM, bool MUL_IR>
__device__ __forceinline__ int place(int u, int i, int mul, int dim) { return MUL_IR ? u * (DIM ? DIM : dim) + i : i * mul + u; }
// how many channels a lane takes at a time
template <int DIM> constexpr int kUnrolled = DIM == 1 ? 4 : DIM == 3 ? 2 : 1;
#define CUEQ_CHANNELS _Pragma("unroll (kUnrolled<DIM>)") for (int u = c.lane; u < c.mul; u += 32)
#define CUEQ_COMPONENTS _Pragma("unroll") for (int i = 0; i < (DIM ? DIM : c.dim); ++i)
#define CUEQ_AT place<DIM, MUL_IR>(u, i, c.mul, c.dim)

template <class T, class M, int MODE, bool Q8, int DIM, bool MUL_IR>
__device__ __forceinline__ void forward_item(const View<M>& c, T* __restrict__ x, T* __restrict__ y, const T* __restrict__ g, signed char* __restrict__ ca,
                                             signed char* __restrict__ cg, signed char* __restrict__ ch, M* __restrict__ stats) {
  const M *__restrict__ cs = c.s, *__restrict__ cw = c.w;
  M* __restrict__ cc = c.a;
  constexpr bool kHasBranch = (MODE & kBranch) != 0;
  const T* t = kHasBranch ? y : x;                       // what the first statistic is of
  M sum = M(0);
  unsigned top = 0, gtop = 0;
  CUEQ_CHANNELS {
    CUEQ_COMPONENTS {
      const M v = to<M>(t[CUEQ_AT]);
      sum += v * v;
      if (Q8) top = max(top, magnitude(v));
    }
    if (Q8 && kHasBranch && c.gated) gtop = max(gtop, magnitude(to<M>(g[u])));
  }
  sum = cueq::warp_sum(sum);
  const M r = inverse_sqrt(sum * c.inv_n + c.eps);
  float step = 0.f, inv = 0.f, gstep = 0.f, ginv = 0.f;
  if (Q8) {
    code_step(__reduce_max_sync(0xffffffffu, top), step, inv);
    if (kHasBranch && c.gated) code_step(__reduce_max_sync(0xffffffffu, gtop), gstep, ginv);
  }
  if (MODE == kNorm) {
    CUEQ_CHANNELS {
      const M a = cw[u] * r;
      CUEQ_COMPONENTS {
        const M v = to<M>(x[CUEQ_AT]);
        if (Q8) ca[CUEQ_AT] = to_code(v, inv);
        x[CUEQ_AT] = from<T>(a * v);
      }
    }
    if (stats && c.lane == 0) { stats[0] = r; stats[2] = M(step); }
    return;
  }
  M hsum = M(0);
  unsigned htop = 0;
  CUEQ_CHANNELS {
    M v = M(1), dv;
    if (c.gated) {
      const M gate = to<M>(g[u]);
      activation<T>(c.gate, gate, v, dv);
      if (Q8) cg[u] = to_code(gate, ginv);
    }
    const M a = cs[u] * v * r;
    if (MODE == kBoth) cc[u] = a;
    CUEQ_COMPONENTS {
      const M yv = to<M>(y[CUEQ_AT]);
      const M h = to<M>(x[CUEQ_AT]) + a * yv;
      if (Q8) ca[CUEQ_AT] = to_code(yv, inv);
      if (MODE == kBranch) x[CUEQ_AT] = from<T>(h);
      else {
        hsum += h * h;
        if (Q8) htop = max(htop, magnitude(h));
      }
    }
  }
  M rh = M(0);
  float hstep = 0.f, hinv = 0.f;
  if (MODE == kBoth) {
    hsum = cueq::warp_sum(hsum);
    rh = inverse_sqrt(hsum * c.inv_n + c.eps);
    if (Q8) code_step(__reduce_max_sync(0xffffffffu, htop), hstep, hinv);
    // h once more from x and y: kept in 16 bits in between, n would be rounded twice
    CUEQ_CHANNELS {
      const M a = cc[u], b = cw[u] * rh;
      CUEQ_COMPONENTS {
        const M h = to<M>(x[CUEQ_AT]) + a * to<M>(y[CUEQ_AT]);
        if (Q8) ch[CUEQ_AT] = to_code(h, hinv);
        x[CUEQ_AT] = from<T>(h);
        y[CUEQ_AT] = from<T>(b * h);
      }
    }
  }
  if (stats && c.lane == 0) {
    stats[0] = r; stats[1] = rh; stats[2] = M(step); stats[3] = M(gstep);
    if (Q8 && MODE == kBoth) stats[4] = M(hstep);
  }
}

// h of the norm behind a branch is formed again from x (in its place), y and the gates
template <class T, class M, int MODE, bool Q8> constexpr bool kAgain = MODE == kBoth && !Q8 && sizeof(T) < sizeof(M);

// K: type of what was kept (T or codes).  r (r c) stays in range: r^2 <= 1 / eps, and r >= 5e-20 while the sum of squares is finite.
template <class T, class M, class K, int MODE, bool Q8, int DIM, bool MUL_IR>
__device__ __forceinline__ void backward_item(const View<M>& c, T* __restrict__ go, T* __restrict__ gn, const K* __restrict__ h, const K* __restrict__ y, const K* g, T* dg,
                                              const M* __restrict__ stats, bool has_go) {
  const M *__restrict__ cs = c.s, *__restrict__ cw = c.w;
  M *__restrict__ cc = c.a, *__restrict__ acc_s = c.acc_s, *__restrict__ acc_w = c.acc_w;
  M rh = M(0), qh = M(0);
  // channel u, element `at` of what was normalised
  auto normed = [&](int u, int at) { return kAgain<T, M, MODE, Q8> ? to<M>(h[at]) + cc[u] * to<M>(y[at]) : to<M>(h[at]); };
  if (MODE & kNorm) {
    rh = stats[MODE == kBoth ? 1 : 0];
    const M step = Q8 ? stats[MODE == kBoth ? 4 : 2] : M(1);
    const M rs = rh * step;
    M dot = M(0);
    CUEQ_CHANNELS {
      if (kAgain<T, M, MODE, Q8>) {
        M v = M(1), dv;
        if (c.gated) activation<T>(c.gate, to<M>(g[u]), v, dv);
        cc[u] = cs[u] * v * stats[0];
      }
      M p = M(0);
      CUEQ_COMPONENTS p += to<M>(gn[CUEQ_AT]) * normed(u, CUEQ_AT);
      p *= rs;
      acc_w[u] += p;
      dot += cw[u] * p;
    }
    qh = rh * (rh * (c.inv_n * cueq::warp_sum(dot))) * step;
    if (MODE == kNorm) {
      CUEQ_CHANNELS {
        const M a = cw[u] * rh;
        CUEQ_COMPONENTS gn[CUEQ_AT] = from<T>(a * to<M>(gn[CUEQ_AT]) - qh * to<M>(h[CUEQ_AT]));
      }
      return;
    }
  }
  // in 32 and 64 bits what reaches h is put down once, over go; in 16 bits it is computed twice, so that dy is rounded once
  constexpr bool kPut = MODE == kBoth && sizeof(T) == sizeof(M);
  const M r = stats[0], step = Q8 ? stats[2] : M(1), gstep = Q8 ? stats[3] : M(1), rs = r * step;
  M dot = M(0);
  CUEQ_CHANNELS {
    M v = M(1), dv = M(0), p = M(0);
    if (c.gated) activation<T>(c.gate, to<M>(g[u]) * gstep, v, dv);
    const M b = MODE == kBoth ? cw[u] * rh : M(0), s = cs[u];
    CUEQ_COMPONENTS {
      M o = MODE == kBranch || has_go ? to<M>(go[CUEQ_AT]) : M(0);
      if (MODE == kBoth) o += b * to<M>(gn[CUEQ_AT]) - qh * normed(u, CUEQ_AT);
      if (kPut) go[CUEQ_AT] = from<T>(o);
      p += o * to<M>(y[CUEQ_AT]);
    }
    p *= rs;
    const M a = s * v;
    cc[u] = a * r;
    acc_s[u] += v * p;
    dot += a * p;
    if (c.gated) dg[u] = from<T>(s * dv * p);            // may lie over g[u]
  }
  const M q = r * (r * (c.inv_n * cueq::warp_sum(dot))) * step;
  CUEQ_CHANNELS {
    const M a = cc[u], b = MODE == kBoth ? cw[u] * rh : M(0);
    CUEQ_COMPONENTS {
      M o = kPut || MODE == kBranch || has_go ? to<M>(go[CUEQ_AT]) : M(0);
      if (MODE == kBoth && !kPut) o += b * to<M>(gn[CUEQ_AT]) - qh * normed(u, CUEQ_AT);
      const T dy = from<T>(a * o - q * to<M>(y[CUEQ_AT]));
      if (MODE == kBoth && !kPut) go[CUEQ_AT] = from<T>(o);
      (MODE == kBoth ? gn : go)[CUEQ_AT] = dy;
    }
  }
}

// ---- rows of an irrep block whose values a warp holds in registers ------------------------------------------------------------------------
// A lane owns K = 1, 2 or 4 neighbouring channels: K * DIM values, moved as DIM vectors of K values in either layout (mul_ir: one behind the
// other; no bank conflicts, DIM is odd).  Shared memory is read once and written once, an instruction for K values.
//
// Short blocks take several rows at a time, as what a call costs besides its values, above all the sums over the warp, is most of their
// time: R rows per lane, or (NARROW, up to 16 channels) a row per `lanes` lanes.  Of missing rows and channels the last one is read instead.
template <int DIM, int K> constexpr int kRowsAtOnce = DIM * K <= 2 ? 4 : DIM == 3 && K <= 2 ? 2 : 1;

// rows of one region: E at byte `base`, `pitch` bytes apart
template <class E>
struct Rows {
  unsigned char* base;
  int pitch;
  __device__ __forceinline__ E* operator[](int q) const { return reinterpret_cast<E*>(base + q * pitch); }
};
template <class E, int K>
struct alignas(sizeof(E) * K < 16 ? sizeof(E) * K : 16) Vec { E v[K]; };

// sums of R values each over the warp, every one by the same pairs in the same order as cueq::warp_sum; NARROW: over `lanes` lanes
template <bool NARROW, int R, class M>
__device__ __forceinline__ void warp_sums(M (&s)[R], int lane, int lanes) {
  constexpr unsigned all = 0xffffffffu;
  if constexpr (NARROW) {
    for (int o = lanes >> 1; o; o >>= 1) s[0] += __shfl_xor_sync(all, s[0], o);
  } else if constexpr (R == 1) {
    s[0] = cueq::warp_sum(s[0]);
  } else {
    M t;
    if constexpr (R == 2) {
      const bool up = lane & 16;
      t = (up ? s[1] : s[0]) + __shfl_xor_sync(all, up ? s[0] : s[1], 16);
      t += __shfl_xor_sync(all, t, 8);
    } else {
      const bool up = lane & 16, odd = lane & 8;
      const M a = (up ? s[1] : s[0]) + __shfl_xor_sync(all, up ? s[0] : s[1], 16), b = (up ? s[3] : s[2]) + __shfl_xor_sync(all, up ? s[2] : s[3], 16);
      t = (odd ? b : a) + __shfl_xor_sync(all, odd ? a : b, 8);
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) t += __shfl_xor_sync(all, t, o);
#pragma unroll
    for (int q = 0; q < R; ++q) s[q] = __shfl_sync(all, t, (q & 1) * 16 + (q >> 1) * 8);
  }
}
template <bool NARROW>
__device__ __forceinline__ unsigned warp_top(unsigned v, int lanes) {
  if constexpr (NARROW) {
    for (int o = lanes >> 1; o; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  } else {
    return __reduce_max_sync(0xffffffffu, v);
  }
}

template <class T, class M, int DIM, bool MUL_IR, int K, int R, bool NARROW>
struct Short {
  int lane, lanes, first, mul, left; // first: this lane's vector of channels; left: rows that there are, from 1 on
  int group;                         // NARROW: this lane's row
  bool on;                           // the lane has channels
  __device__ __forceinline__ Short(const View<M>& c, int left_) : lane(c.lane), lanes(c.lanes), mul(c.mul), left(left_) {
    const int l = NARROW ? lane % lanes : lane;
    group = NARROW ? lane / lanes : 0;
    on = l * K < mul;
    first = on ? l : 0;
  }
  __device__ __forceinline__ int row(int q) const { return NARROW ? min(group, left - 1) : R == 1 ? 0 : min(q, left - 1); }
  __device__ __forceinline__ bool there(int q) const { return on && (NARROW ? group < left : R == 1 || q < left); }
  // vector j of DIM, in vectors
  __device__ __forceinline__ int at(int j) const { return MUL_IR ? first * DIM + j : j * (mul / K) + first; }
  template <class E>
  __device__ __forceinline__ void load(const Rows<E>& p, M (&v)[R][K][DIM]) const {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const Vec<E, K>* e = reinterpret_cast<const Vec<E, K>*>(p[row(q)]);
#pragma unroll
      for (int j = 0; j < DIM; ++j) {
        const Vec<E, K> x = e[at(j)];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (MUL_IR) v[q][(j * K + k) / DIM][(j * K + k) % DIM] = to<M>(x.v[k]);
          else v[q][k][j] = to<M>(x.v[k]);
        }
      }
    }
  }
  // v += a times a row of values, one factor per channel
  template <class E>
  __device__ __forceinline__ void add_scaled(const E* row, const M (&a)[K], M (&v)[K][DIM]) const {
    const Vec<E, K>* e = reinterpret_cast<const Vec<E, K>*>(row);
#pragma unroll
    for (int j = 0; j < DIM; ++j) {
      const Vec<E, K> x = e[at(j)];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (MUL_IR) v[(j * K + k) / DIM][(j * K + k) % DIM] += a[(j * K + k) / DIM] * to<M>(x.v[k]);
        else v[k][j] += a[k] * to<M>(x.v[k]);
      }
    }
  }
  template <class E, class F>
  __device__ __forceinline__ void put(E* row, const M (&v)[K][DIM], F convert) const {
    Vec<E, K>* e = reinterpret_cast<Vec<E, K>*>(row);
#pragma unroll
    for (int j = 0; j < DIM; ++j) {
      Vec<E, K> x;
#pragma unroll
      for (int k = 0; k < K; ++k) x.v[k] = convert(MUL_IR ? v[(j * K + k) / DIM][(j * K + k) % DIM] : v[k][j]);
      e[at(j)] = x;
    }
  }
  __device__ __forceinline__ void store(const Rows<T>& p, const M (&v)[R][K][DIM]) const {
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (there(q)) put(p[row(q)], v[q], [](M m) { return from<T>(m); });
  }
  // K values of a row of channels
  template <class E>
  __device__ __forceinline__ void channels(const E* row, M (&v)[K]) const {
    const Vec<E, K> x = reinterpret_cast<const Vec<E, K>*>(row)[first];
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = to<M>(x.v[k]);
  }
  template <class E, class F>
  __device__ __forceinline__ void put_channels(E* row, const M (&v)[K], F convert) const {
    Vec<E, K> x;
#pragma unroll
    for (int k = 0; k < K; ++k) x.v[k] = convert(v[k]);
    reinterpret_cast<Vec<E, K>*>(row)[first] = x;
  }
  // this lane's sums of its channels, one set per lane (NARROW) or channel
  __device__ __forceinline__ void add(M* sums, const M (&v)[K]) const {
    if (!on) return;
    Vec<M, K>* e = reinterpret_cast<Vec<M, K>*>(sums) + (NARROW ? lane : first);
    Vec<M, K> x = *e;
#pragma unroll
    for (int k = 0; k < K; ++k) x.v[k] += v[k];
    *e = x;
  }
  // steps of the rows, and their codes
  __device__ __forceinline__ void code(const Rows<signed char>& p, const M (&v)[R][K][DIM], float (&step)[R]) const {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      unsigned t = 0;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < DIM; ++i) t = max(t, magnitude(v[q][k][i]));
      float inverse;
      code_step(warp_top<NARROW>(t, lanes), step[q], inverse);
      if (there(q)) put(p[row(q)], v[q], [=](M m) { return to_code(m, inverse); });
    }
  }
  // r of the rows
  __device__ __forceinline__ void inverse_rms(const M (&v)[R][K][DIM], M inv_n, M eps, M (&r)[R]) const {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      M part[DIM];
#pragma unroll
      for (int i = 0; i < DIM; ++i) part[i] = v[q][0][i] * v[q][0][i];
#pragma unroll
      for (int k = 1; k < K; ++k)
#pragma unroll
        for (int i = 0; i < DIM; ++i) part[i] += v[q][k][i] * v[q][k][i];
#pragma unroll
      for (int i = 1; i < DIM; ++i) part[0] += part[i];
      r[q] = on ? part[0] : M(0);
    }
    warp_sums<NARROW>(r, lane, lanes);
#pragma unroll
    for (int q = 0; q < R; ++q) r[q] = inverse_sqrt(r[q] * inv_n + eps);
  }
  __device__ __forceinline__ bool leads() const { return NARROW ? lane % lanes == 0 : lane == 0; }
};

template <class T, class M, int MODE, bool Q8, int DIM, bool MUL_IR, int K, int R, bool NARROW>
__device__ __forceinline__ void forward_short(const View<M>& c, int left, Rows<T> x, Rows<T> y, Rows<T> g, Rows<signed char> ca, Rows<signed char> cg,
                                              Rows<signed char> ch, M* stats, int64_t ld_stats) {
  const Short<T, M, DIM, MUL_IR, K, R, NARROW> w(c, left);
  M v[R][K][DIM], xv[R][K][DIM], a[R][K], r[R], rh[R], s[K];
  float step[R], gstep[R], hstep[R];
  w.load((MODE & kBranch) ? y : x, v);
  if (MODE & kBranch) w.load(x, xv);
  w.channels((MODE & kBranch) ? c.s : c.w, s);
#pragma unroll
  for (int q = 0; q < R; ++q) {
    gstep[q] = 0.f;
    if ((MODE & kBranch) && c.gated) {
      M gate[K];
      w.channels(g[w.row(q)], gate);
      if (Q8) {
        unsigned top = 0;
        float inverse;
#pragma unroll
        for (int k = 0; k < K; ++k) top = max(top, magnitude(gate[k]));
        code_step(warp_top<NARROW>(top, w.lanes), gstep[q], inverse);
        if (w.there(q)) w.put_channels(cg[w.row(q)], gate, [=](M m) { return to_code(m, inverse); });
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        M e, de;
        activation<T>(c.gate, gate[k], e, de);
        a[q][k] = s[k] * e;
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) a[q][k] = s[k];
    }
  }
  w.inverse_rms(v, c.inv_n, c.eps, r);
  if (Q8) w.code(ca, v, step);
#pragma unroll
  for (int q = 0; q < R; ++q)
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < DIM; ++i) v[q][k][i] = (MODE & kBranch) ? xv[q][k][i] + a[q][k] * r[q] * v[q][k][i] : a[q][k] * r[q] * v[q][k][i];
  w.store(x, v);
  if (MODE == kBoth) {
    w.inverse_rms(v, c.inv_n, c.eps, rh);
    if (Q8) w.code(ch, v, hstep);
    w.channels(c.w, s);
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < DIM; ++i) v[q][k][i] *= s[k] * rh[q];
    w.store(y, v);
  }
  if (stats && w.leads()) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (!w.there(q)) break;
      M* e = stats + w.row(q) * ld_stats;
      e[0] = r[q];
      if (MODE == kBoth) e[1] = rh[q];
      if (Q8) { e[2] = M(step[q]); e[3] = M(gstep[q]); }
      if (Q8 && MODE == kBoth) e[4] = M(hstep[q]);
    }
  }
}

template <class T, class M, class K8, int MODE, bool Q8, int DIM, bool MUL_IR, int K, int R, bool NARROW>
__device__ __forceinline__ void backward_short(const View<M>& c, int left, Rows<T> go, Rows<T> gn, Rows<K8> h, Rows<K8> y, Rows<K8> g, Rows<T> dg,
                                               Rows<M> stats, bool has_go) {
  const Short<T, M, DIM, MUL_IR, K, R, NARROW> w(c, left);
  constexpr bool again = kAgain<T, M, MODE, Q8>;
  M o[R][K][DIM], v[R][K][DIM], dot[R], sum[K], s[K];
  M act[R][K], dact[R][K];                               // again: kept from one use to the other (computed twice: 311 us for 217 with 128x(0e+1o+2e+3o))
  if (MODE & kNorm) {
    M rh[R], step[R], b[K];
    w.load(gn, o);
    w.load(h, v);
    if constexpr (again) {                               // v is x
      w.channels(c.s, s);
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const M r1 = stats[w.row(q)][0];
        M gate[K], ar[K];
        if (c.gated) w.channels(g[w.row(q)], gate);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          M e = M(1), de = M(0);
          if (c.gated) activation<T>(c.gate, gate[k], e, de);
          act[q][k] = e; dact[q][k] = de;
          ar[k] = s[k] * e * r1;
        }
        w.add_scaled(y[w.row(q)], ar, v[q]);
      }
    }
    w.channels(c.w, b);
#pragma unroll
    for (int k = 0; k < K; ++k) sum[k] = M(0);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const M* e = stats[w.row(q)];
      rh[q] = e[MODE == kBoth ? 1 : 0];
      step[q] = Q8 ? e[MODE == kBoth ? 4 : 2] : M(1);
      dot[q] = M(0);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        M p = M(0);
#pragma unroll
        for (int i = 0; i < DIM; ++i) p += o[q][k][i] * v[q][k][i];
        p *= rh[q] * step[q];
        sum[k] += w.there(q) ? p : M(0);
        dot[q] += b[k] * p;
      }
      dot[q] = w.on ? dot[q] : M(0);
    }
    w.add(c.acc_w, sum);
    warp_sums<NARROW>(dot, c.lane, w.lanes);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const M qh = rh[q] * (rh[q] * (c.inv_n * dot[q])) * step[q];
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < DIM; ++i) o[q][k][i] = b[k] * rh[q] * o[q][k][i] - qh * v[q][k][i];
    }
    if (MODE == kNorm) {
      w.store(gn, o);
      return;
    }
    if (has_go) {
      w.load(go, v);
#pragma unroll
      for (int q = 0; q < R; ++q)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < DIM; ++i) o[q][k][i] += v[q][k][i];
    }
    w.store(go, o);
  } else {
    w.load(go, o);
  }
  M r[R], step[R], a[R][K];
  w.load(y, v);
  if (!again) w.channels(c.s, s);
#pragma unroll
  for (int k = 0; k < K; ++k) sum[k] = M(0);
#pragma unroll
  for (int q = 0; q < R; ++q) {
    const M* st = stats[w.row(q)];
    r[q] = st[0];
    step[q] = Q8 ? st[2] : M(1);
    dot[q] = M(0);
    M gate[K], de[K];
    if (c.gated && !again) w.channels(g[w.row(q)], gate);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      M e = M(1), p = M(0);
      de[k] = M(0);
      if constexpr (again) { e = act[q][k]; de[k] = dact[q][k]; }
      else if (c.gated) activation<T>(c.gate, Q8 ? gate[k] * st[3] : gate[k], e, de[k]);
#pragma unroll
      for (int i = 0; i < DIM; ++i) p += o[q][k][i] * v[q][k][i];
      p *= r[q] * step[q];
      a[q][k] = s[k] * e;
      dot[q] += a[q][k] * p;
      sum[k] += w.there(q) ? e * p : M(0);
      de[k] *= s[k] * p;
    }
    dot[q] = w.on ? dot[q] : M(0);
    if (c.gated && w.there(q)) w.put_channels(dg[w.row(q)], de, [](M m) { return from<T>(m); });   // may lie over g, of which no other lane reads this
  }
  w.add(c.acc_s, sum);
  warp_sums<NARROW>(dot, c.lane, w.lanes);
#pragma unroll
  for (int q = 0; q < R; ++q) {
    const M qy = r[q] * (r[q] * (c.inv_n * dot[q])) * step[q];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < DIM; ++i) v[q][k][i] = a[q][k] * r[q] * o[q][k][i] - qy * v[q][k][i];
  }
  w.store(MODE == kBoth ? gn : go, v);
}

// ---- moving rows ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bulk_in(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
               ::"r"(s32(dst)), "l"(src), "r"(bytes), "r"(s32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_out(void* dst, const void* src, unsigned bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(dst), "r"(s32(src)), "r"(bytes) : "memory");
}

// A tensor's rows in memory and their region; elements of `size` bytes (codes and statistics: 16).  The last stage of a dense tensor may hold
// bytes behind the last 16: these move like kPlain.
struct Move { Region reg; int size, route; unsigned char* mem; int64_t ld; };

template <bool IN, class E>
__device__ __forceinline__ void copy_elements(unsigned char* smem, unsigned char* mem, int from, int bytes, int lane) {
  E *a = reinterpret_cast<E*>(smem), *b = reinterpret_cast<E*>(mem);
  for (int e = from / (int)sizeof(E) + lane; e < bytes / (int)sizeof(E); e += 32) {
    if (IN) a[e] = __ldg(b + e); else b[e] = a[e];
  }
}
template <bool IN>
__device__ __forceinline__ void copy_row(unsigned char* smem, unsigned char* mem, int from, int bytes, int size, int lane) {
  switch (size) {
    case 2: copy_elements<IN, unsigned short>(smem, mem, from, bytes, lane); break;
    case 4: copy_elements<IN, unsigned>(smem, mem, from, bytes, lane); break;
    case 8: copy_elements<IN, unsigned long long>(smem, mem, from, bytes, lane); break;
    default: copy_elements<IN, uint4>(smem, mem, from, bytes, lane); break;
  }
}
template <bool IN>
__device__ __noinline__ void copy_rest(const Move* moves, int count, unsigned char* stage, int64_t z, int n) {
  const int lane = threadIdx.x;
  for (int k = 0; k < count; ++k) {
    const Move& m = moves[k];
    unsigned char *a = stage + m.reg.at, *b = m.mem + z * m.ld;
    if (m.route == kPlain) for (int r = 0; r < n; ++r) copy_row<IN>(a + r * m.reg.pitch, b + r * m.ld, 0, m.reg.bytes, m.size, lane);
    if (m.route == kDense) copy_row<IN>(a, b, n * m.reg.bytes & ~15, n * m.reg.bytes, m.size, lane);
  }
}

// The bulk copy that a lane issues per stage: one row of one tensor, or all rows of a dense one.
static_assert(sizeof(Move) == kMoveBytes, "moves have their room in front of the stages");
struct Job {
  unsigned at;                       // inside a stage
  int bytes, row;                    // of a row; a dense tensor: row = -1
  unsigned char* mem;                // in the next stage
  int64_t step;                      // from stage to stage
  bool rest;                         // some tensor needs copy_rest
};
__device__ __forceinline__ Job make_job(const Move* moves, int count, int rps, int64_t first) {
  Job j{0u, 0, 0, nullptr, 0, false};
  int at = 0;
  for (int k = 0; k < count; ++k) {
    const Move& m = moves[k];
    if (m.route == kPlain) { j.rest = true; continue; }
    const int lanes = m.route == kDense ? 1 : rps, r = (int)threadIdx.x - at;
    if (r >= 0 && r < lanes) {
      j.at = m.reg.at + r * m.reg.pitch;
      j.bytes = m.reg.bytes;
      j.row = m.route == kDense ? -1 : r;
      j.mem = m.mem + (first + r) * m.ld;
      j.step = rps * m.ld;
    }
    at += lanes;
  }
  return j;
}
// bytes that this lane's copy has with n rows in the stage
__device__ __forceinline__ unsigned job_bytes(const Job& j, int n) { return j.row < 0 ? (unsigned)(n * j.bytes) & ~15u : j.row < n ? j.bytes : 0u; }

// Rows first .. last in stages of rps rows; `work(stage, z, n)`.  A lane that issues loads into a stage waits for its own stores out of
// it; the warp then meets, so that no lane's load overtakes another lane's store.  Or one stage at a time.
// `ready()` runs while the first loads are under way.  `phases`, bit s: the phase that stage s waits for.  False: given up.
template <class Ready, class Work>
__device__ __forceinline__ bool run_stages(const Params& p, int rps, int64_t first, int64_t last, const Move* in, int nin, const Move* out, int nout,
                                           unsigned char* stages, int stage_bytes, unsigned long long* full, unsigned& phases, Ready ready, Work work) {
  const int lane = threadIdx.x;
  Job jin = make_job(in, nin, rps, first), jout = make_job(out, nout, rps, first);
  auto load = [&](int64_t z, int s) {
    const int n = (int)min((int64_t)rps, last - z);
    unsigned char* stage = stages + s * stage_bytes;
    const unsigned bytes = job_bytes(jin, n), sum = __reduce_add_sync(0xffffffffu, bytes);
    if (lane == 0) bar_expect_tx(full + s, sum);         // none: the arrival alone completes the phase
    __syncwarp();
    if (bytes) bulk_in(stage + jin.at, jin.mem, bytes, full + s);
    jin.mem += jin.step;
    if (jin.rest || n < rps) {
      copy_rest<true>(in, nin, stage, z, n);
      __syncwarp();                                      // other lanes read what this one has stored; neither a vote nor the barrier orders that
    }
  };
  const bool two = p.stages == 2;
  if (first < last) load(first, 0);
  ready();
  int s = 0;
  for (int64_t z = first; z < last; z += rps) {
    const int n = (int)min((int64_t)rps, last - z);
    const bool more = z + rps < last;
    if (two && more) {
      asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
      __syncwarp();
      load(z + rps, s ^ 1);
    }
    if (!__all_sync(0xffffffffu, bar_wait(full + s, phases >> s & 1, p.status))) {   // a copy did not arrive in time: give up once those in flight have landed
      if (two && more) bar_wait(full + (s ^ 1), phases >> (s ^ 1) & 1, p.status);
      bar_wait(full + s, phases >> s & 1, p.status);
      asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
      return false;
    }
    phases ^= 1u << s;
    unsigned char* stage = stages + s * stage_bytes;
    work(stage, z, n);
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncwarp();
    const unsigned bytes = job_bytes(jout, n);
    if (bytes) bulk_out(jout.mem, stage + jout.at, bytes);
    asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
    jout.mem += jout.step;
    if (jout.rest || n < rps) copy_rest<false>(out, nout, stage, z, n);
    if (two) s ^= 1;
    else if (more) {
      asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
      __syncwarp();
      load(z + rps, 0);
    }
  }
  asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory");
  __syncwarp();
  return true;
}

// The units of rows that this warp takes of each slice.  They are dealt out row by row, all slices of one before the next, in equal numbers: every
// warp has its share of every slice, whatever a slice costs.
struct Share {
  int64_t a, b;                      // units of the first slice; of slice s one more where s lies before `ra`, `rb`
  int ra, rb;
  __device__ __forceinline__ explicit Share(const Params& p) {
    const int64_t j = blockIdx.x, from = j * p.deal + min(j, (int64_t)p.deal_more), to = from + p.deal + (j < p.deal_more ? 1 : 0);
    a = divide(from, p.num_slices, ra);
    b = divide(to, p.num_slices, rb);
  }
  static __device__ __forceinline__ int64_t divide(int64_t v, int n, int& rest) {
    if (n == 1) { rest = 0; return v; }
    const int64_t q = v < 0x7fffffff ? (int64_t)((unsigned)v / (unsigned)n) : v / n;
    rest = (int)(v - q * n);
    return q;
  }
  __device__ __forceinline__ void rows(const Params& p, int s, int64_t& first, int64_t& last) const {
    first = (a + (s < ra)) * p.unit;
    last = min(p.rows, (b + (s < rb)) * p.unit);
  }
};
__device__ __forceinline__ void init_barriers(unsigned char* smem) {
  if (threadIdx.x == 0) {
    bar_init(reinterpret_cast<unsigned long long*>(smem), 1);
    bar_init(reinterpret_cast<unsigned long long*>(smem) + 1, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
}
// parameters of the slice's channels into shared memory, sums cleared
template <class M, int MODE, bool BACKWARD>
__device__ __forceinline__ void prepare(const Params& p, const Slice& s, M* at) {
  const int ch = p.blk[s.first].ch;
  const Head h = head_of(s, MODE, BACKWARD);
  // 128 channels at a time: all loads before the first store
  auto fill = [&](auto load) {
    for (int u = threadIdx.x; u < s.channels; u += 128) {
      M vs[4], vw[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int v = min(u + 32 * q, s.channels - 1);
        if (MODE & kBranch) vs[q] = load(p.s, ch + v);
        if (MODE & kNorm) vw[q] = load(p.w, ch + v);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (u + 32 * q < s.channels) {
          if (MODE & kBranch) at[h.s + u + 32 * q] = vs[q];
          if (MODE & kNorm) at[h.w + u + 32 * q] = vw[q];
        }
    }
  };
  if (p.pdtype == (sizeof(M) == 8 ? CUEQ_F64 : CUEQ_F32)) fill([](const void* q, int i) { return __ldg(reinterpret_cast<const M*>(q) + i); });
  else fill([&](const void* q, int i) { return cueq::load_as<M>(q, p.pdtype, i); });
  for (int u = h.sum_s + threadIdx.x; u < h.total; u += 32) at[u] = M(0);
  __syncwarp();
}
template <class M, int MODE, bool BACKWARD>
__device__ __forceinline__ View<M> block_view(const Params& p, const Slice& s, const Blk& b, M* at) {
  View<M> c;
  const int u0 = b.ch - p.blk[s.first].ch;
  const Head h = head_of(s, MODE, BACKWARD);
  c.s = at + h.s + u0; c.w = at + h.w + u0; c.a = at + h.a + u0; c.acc_s = at + h.sum_s + b.sum; c.acc_w = at + h.sum_w + b.sum;
  c.mul = b.mul; c.dim = b.dim;
  c.lane = threadIdx.x; c.lanes = b.lanes;
  c.gate = p.gate; c.gated = p.gate != CUEQ_NORM_GATE_NONE;
  c.inv_n = reciprocal(M(b.mul * b.dim));
  c.eps = M(p.eps);
  return c;
}

template <int NIN, int NOUT>
__device__ __forceinline__ void put_moves(Move* moves, const Move (&in)[NIN], int nin, const Move (&out)[NOUT], int nout) {
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 0; k < NIN; ++k) if (k < nin) moves[k] = in[k];
#pragma unroll
    for (int k = 0; k < NOUT; ++k) if (k < nout) moves[nin + k] = out[k];
  }
  __syncwarp();
}

// (dimension, channels per lane) of a block: SHORT for those that registers hold, LONG, row by row, for the others
#define CUEQ_NORM_K(D, SHORT)                                                          \
  if (b.per_lane == 4) { SHORT(D, 4) }                                                 \
  else if (b.per_lane == 2) { SHORT(D, 2) }                                            \
  else { SHORT(D, 1) }
#define CUEQ_NORM_DIMS(SHORT, LONG)                                                    \
  if (b.per_lane) {                                                                    \
    switch (b.dim) {                                                                   \
      case 1: CUEQ_NORM_K(1, SHORT) break;                                             \
      case 3: CUEQ_NORM_K(3, SHORT) break;                                             \
      case 5: CUEQ_NORM_K(5, SHORT) break;                                             \
      default: CUEQ_NORM_K(7, SHORT) break;                                            \
    }                                                                                  \
  } else {                                                                             \
    switch (b.dim) {                                                                   \
      case 1: LONG(1) break;                                                           \
      case 3: LONG(3) break;                                                           \
      case 5: LONG(5) break;                                                           \
      case 7: LONG(7) break;                                                           \
      default: LONG(0) break;                                                          \
    }                                                                                  \
  }
// one row at a time, several per lane, or several side by side
#define CUEQ_SHORT(D, N)                                                                                               \
  if (N == 1 && b.lanes < 32) { CUEQ_ROWS(D, 1, 1, true, 32 / b.lanes) }                                               \
  else if (kRowsAtOnce<D, N> > 1 && n > 1) { CUEQ_ROWS(D, N, (kRowsAtOnce<D, N>), false, (kRowsAtOnce<D, N>)) }        \
  else { CUEQ_ROWS(D, N, 1, false, 1) }

template <class T, class M, int MODE, bool Q8, bool MUL_IR>
__device__ __forceinline__ bool forward_slice(const Params& p, const Slice& sl, int64_t first, int64_t last, unsigned char* smem, unsigned& phases) {
  M* at = reinterpret_cast<M*>(smem + kBars);
  constexpr int size = sizeof(T);
  const Stage st = forward_stage(p, sl, MODE, Q8, size);
  const Blk& b0 = p.blk[sl.first];
  const bool gated = (MODE & kBranch) && p.gate != CUEQ_NORM_GATE_NONE;
  auto ptr = [](const void* q, int64_t bytes) { return reinterpret_cast<unsigned char*>(const_cast<void*>(q)) + bytes; };
  const int64_t fo = (int64_t)b0.off * size, ldo = (int64_t)p.dim_total * size;
  Move* moves = reinterpret_cast<Move*>(smem + 16);
  const Move in[3] = {{st.a, size, p.route[tX], ptr(p.x, fo), p.ldx * size},
                      {st.b, size, p.route[tY], ptr(p.y, fo), p.ldy * size},
                      {st.g, size, p.route[tG], ptr(p.g, (int64_t)b0.ch * size), p.ldg * size}};
  const Move o_first = {st.a, size, p.route[(MODE & kBranch) ? tOut : tNorm], ptr((MODE & kBranch) ? p.out : p.norm, fo), ldo};
  const Move o_norm = {st.b, size, p.route[tNorm], ptr(p.norm, fo), ldo};
  const Move o_ca = {st.ca, 16, kRows, (unsigned char*)p.codes + b0.code, p.ldc};
  const Move o_cg = {st.cg, 16, kRows, (unsigned char*)p.codes + b0.gcode, p.ldc};
  const Move o_ch = {st.ch, 16, kRows, (unsigned char*)p.codes + b0.hcode, p.ldc};
  // those that a call does not have come last
  const Move out[5] = {o_first, MODE == kBoth ? o_norm : o_ca, MODE == kBoth ? o_ca : o_cg, MODE == kBoth ? o_ch : o_cg, o_cg};
  const int nout = 1 + (MODE == kBoth) + (Q8 ? 1 + (MODE == kBoth) + gated : 0);
  const int nin = (MODE & kBranch) ? 2 + gated : 1;
  put_moves(moves, in, nin, out, nout);
  return run_stages(p, sl.rps, first, last, moves, nin, moves + nin, nout, smem + head_bytes(sizeof(M), sl, MODE, false), st.total,
                    reinterpret_cast<unsigned long long*>(smem), phases, [&]() { prepare<M, MODE, false>(p, sl, at); }, [&](unsigned char* s, int64_t z, int n) {
    for (int k = sl.first; k < sl.first + sl.count; ++k) {
      const Blk& b = p.blk[k];
      const View<M> c = block_view<M, MODE, false>(p, sl, b, at);
      const int e = b.off - b0.off, u = b.ch - b0.ch;
      auto region = [&](const Region& reg, int bytes) { return s + reg.at + bytes; };
      const Rows<T> rx{region(st.a, e * size), st.a.pitch}, ry{region(st.b, e * size), st.b.pitch}, rg{region(st.g, u * size), st.g.pitch};
      const Rows<signed char> ra{region(st.ca, b.code - b0.code), st.ca.pitch}, rc{region(st.cg, b.gcode - b0.gcode), st.cg.pitch},
          rh{region(st.ch, b.hcode - b0.hcode), st.ch.pitch};
      const int64_t ld_stats = (int64_t)p.nb * p.ns;
      M* stats = p.stats ? reinterpret_cast<M*>(p.stats) + z * ld_stats + k * p.ns : nullptr;
      auto rows_on = [](auto t, int r) { t.base += r * t.pitch; return t; };
#define CUEQ_ROWS(D, N, R, NARROW, STEP)                                                                                                \
  for (int r = 0; r < n; r += STEP)                                                                                                    \
    forward_short<T, M, MODE, Q8, D, MUL_IR, N, R, NARROW>(c, n - r, rows_on(rx, r), rows_on(ry, r), rows_on(rg, r), rows_on(ra, r),     \
                                                           rows_on(rc, r), rows_on(rh, r), stats ? stats + r * ld_stats : nullptr, ld_stats);
#define CUEQ_LONG(D)                                                                                                                   \
  for (int r = 0; r < n; ++r)                                                                                                          \
    forward_item<T, M, MODE, Q8, D, MUL_IR>(c, rx[r], ry[r], rg[r], ra[r], rc[r], rh[r], stats ? stats + r * ld_stats : nullptr);
      CUEQ_NORM_DIMS(CUEQ_SHORT, CUEQ_LONG)
#undef CUEQ_LONG
#undef CUEQ_ROWS
    }
  });
}

template <class T, bool Q8> struct Kept { using type = T; };
template <class T> struct Kept<T, true> { using type = signed char; };

template <class T, class M, int MODE, bool Q8, bool MUL_IR>
__device__ __forceinline__ bool backward_slice(const Params& p, const Slice& sl, int64_t first, int64_t last, unsigned char* smem, unsigned& phases) {
  using K = typename Kept<T, Q8>::type;
  M* at = reinterpret_cast<M*>(smem + kBars);
  constexpr int size = sizeof(T);
  const int stat = p.ns * (int)sizeof(M);
  const Stage st = backward_stage(p, sl, MODE, Q8, size, stat);
  const Blk& b0 = p.blk[sl.first];
  const bool branch = MODE & kBranch, gated = branch && p.gate != CUEQ_NORM_GATE_NONE, has_go = p.go != nullptr;
  auto ptr = [](const void* q, int64_t bytes) { return reinterpret_cast<unsigned char*>(const_cast<void*>(q)) + bytes; };
  const int64_t fo = (int64_t)b0.off * size, uo = (int64_t)b0.ch * size, ldo = (int64_t)p.dim_total * size;
  unsigned char* codes = (unsigned char*)p.codes;
  Move* moves = reinterpret_cast<Move*>(smem + 16);
  const Move i_st = {st.st, 16, p.route[tStats], (unsigned char*)p.stats + (int64_t)sl.first * stat, (int64_t)p.nb * stat};
  const Move i_go = {st.a, size, p.route[tGo], ptr(p.go, fo), p.ldgo * size};
  const Move i_gn = {st.b, size, p.route[tGn], ptr(p.gn, fo), p.ldgn * size};
  const Move i_h = Q8 ? Move{st.c, 16, kRows, codes + (MODE == kBoth ? b0.hcode : b0.code), p.ldc} : Move{st.c, size, p.route[tH], ptr(p.h, fo), p.ldh * size};
  const Move i_y = Q8 ? Move{st.d, 16, kRows, codes + b0.code, p.ldc} : Move{st.d, size, p.route[tY], ptr(p.y, fo), p.ldy * size};
  const Move i_g = Q8 ? Move{st.g, 16, kRows, codes + b0.gcode, p.ldc} : Move{st.g, size, p.route[tG], ptr(p.g, uo), p.ldg * size};
  // those that a call does not have come last
  const Move in[6] = {i_st, branch ? i_y : i_h, branch ? (MODE == kBoth ? i_h : i_go) : i_gn, MODE == kBoth ? i_gn : i_g,
                      MODE == kBoth && gated ? i_g : i_go, i_go};
  const int nin = MODE == kNorm ? 3 : MODE == kBranch ? 3 + gated : 4 + gated + has_go;
  const Move o_a = {st.a, size, p.route[MODE == kBoth ? tDx : tDy], ptr(MODE == kBoth ? p.dx : p.dy, fo), ldo};
  const Move o_b = {st.b, size, p.route[branch ? tDy : tDx], ptr(branch ? p.dy : p.dx, fo), ldo};
  const Move o_g = {st.dg, size, p.route[tDg], ptr(p.dg, uo), (int64_t)p.channels * size};
  const Move out[3] = {MODE == kNorm ? o_b : o_a, MODE == kBoth ? o_b : o_g, o_g};
  const int nout = MODE == kNorm ? 1 : 1 + (MODE == kBoth) + gated;
  put_moves(moves, in, nin, out, nout);
  const bool done = run_stages(p, sl.rps, first, last, moves, nin, moves + nin, nout, smem + head_bytes(sizeof(M), sl, MODE, true), st.total,
                               reinterpret_cast<unsigned long long*>(smem), phases, [&]() { prepare<M, MODE, true>(p, sl, at); }, [&](unsigned char* s, int64_t, int n) {
    for (int k = sl.first; k < sl.first + sl.count; ++k) {
      const Blk& b = p.blk[k];
      const View<M> c = block_view<M, MODE, true>(p, sl, b, at);
      const int e = b.off - b0.off, u = b.ch - b0.ch;
      const int ce = Q8 ? b.code - b0.code : e, he = Q8 ? (MODE == kBoth ? b.hcode - b0.hcode : b.code - b0.code) : e, ge = Q8 ? b.gcode - b0.gcode : u;
      auto region = [&](const Region& reg, int bytes) { return s + reg.at + bytes; };
      const Rows<T> ra{region(st.a, e * size), st.a.pitch}, rb{region(st.b, e * size), st.b.pitch}, rd{region(st.dg, u * size), st.dg.pitch};
      const Rows<K> rh{region(st.c, he * (int)sizeof(K)), st.c.pitch}, ry{region(st.d, ce * (int)sizeof(K)), st.d.pitch},
          rg{region(st.g, ge * (int)sizeof(K)), st.g.pitch};
      const Rows<M> rs{region(st.st, (k - sl.first) * stat), st.st.pitch};
      auto rows_on = [](auto t, int r) { t.base += r * t.pitch; return t; };
#define CUEQ_ROWS(D, N, R, NARROW, STEP)                                                                                                \
  for (int r = 0; r < n; r += STEP)                                                                                                    \
    backward_short<T, M, K, MODE, Q8, D, MUL_IR, N, R, NARROW>(c, n - r, rows_on(ra, r), rows_on(rb, r), rows_on(rh, r), rows_on(ry, r), \
                                                               rows_on(rg, r), rows_on(rd, r), rows_on(rs, r), has_go);
#define CUEQ_LONG(D)                                                                                                                   \
  for (int r = 0; r < n; ++r) backward_item<T, M, K, MODE, Q8, D, MUL_IR>(c, ra[r], rb[r], rh[r], ry[r], rg[r], rd[r], rs[r], has_go);
      CUEQ_NORM_DIMS(CUEQ_SHORT, CUEQ_LONG)
#undef CUEQ_LONG
#undef CUEQ_ROWS
    }
  });
  // this warp's sums of the parameters' gradients
  if (!p.parts) return done;
  M* dst = reinterpret_cast<M*>(p.parts) + (int64_t)blockIdx.x * p.channels + b0.ch;
  const Head head = head_of(sl, MODE, true);
  for (int k = sl.first; k < sl.first + sl.count; ++k) {
    const Blk& b = p.blk[k];
    const M *sums_s = at + head.sum_s + b.sum, *sums_w = at + head.sum_w + b.sum;
    const int groups = b.per_lane == 1 ? 32 / b.lanes : 1;
    for (int u = threadIdx.x; u < b.mul; u += 32) {
      M vs = M(0), vw = M(0);
      for (int g = 0; g < groups; ++g) {
        if (MODE & kBranch) vs += sums_s[g * b.lanes + u];
        if (MODE & kNorm) vw += sums_w[g * b.lanes + u];
      }
      if (MODE & kBranch) dst[b.ch - b0.ch + u] = vs;
      if (MODE & kNorm) dst[(int64_t)gridDim.x * p.channels + b.ch - b0.ch + u] = vw;
    }
  }
  __syncwarp();
  return done;
}

template <class T, class M, int MODE, bool Q8, bool MUL_IR>
__global__ void __launch_bounds__(32, warps_per_sm(sizeof(M))) forward_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  init_barriers(smem);
  unsigned phases = 0;
  const Share share(p);
  int s = blockIdx.x % p.num_slices;                     // neighbouring warps start with different slices
  for (int k = 0; k < p.num_slices; ++k, s = s + 1 == p.num_slices ? 0 : s + 1) {
    int64_t first, last;
    share.rows(p, s, first, last);
    if (first < last && !forward_slice<T, M, MODE, Q8, MUL_IR>(p, p.slice[s], first, last, smem, phases)) return;
  }
}
template <class T, class M, int MODE, bool Q8, bool MUL_IR>
__global__ void __launch_bounds__(32, warps_per_sm(sizeof(M))) backward_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  init_barriers(smem);
  unsigned phases = 0;
  const Share share(p);
  // The warps of an SM work on one slice at a time: the code of four dimensions together does not fit into its instruction cache (186
  // against 201 us for 32,768 rows of 128x(0e+1o+2e+3o) in codes).  The forward code is short enough for all, and faster so.
  int s = blockIdx.x % kSms % p.num_slices;
  for (int k = 0; k < p.num_slices; ++k, s = s + 1 == p.num_slices ? 0 : s + 1) {
    int64_t first, last;
    share.rows(p, s, first, last);
    if (first >= last) {                                 // fewer rows than warps: its sums are nothing
      if (!p.parts) continue;
      const Slice& sl = p.slice[s];
      M* dst = reinterpret_cast<M*>(p.parts) + (int64_t)blockIdx.x * p.channels + p.blk[sl.first].ch;
      for (int u = threadIdx.x; u < sl.channels; u += 32) {
        if (MODE & kBranch) dst[u] = M(0);
        if (MODE & kNorm) dst[(int64_t)gridDim.x * p.channels + u] = M(0);
      }
    } else if (!backward_slice<T, M, MODE, Q8, MUL_IR>(p, p.slice[s], first, last, smem, phases)) return;
  }
}

using Kernel = void (*)(Params);

// the kernels of one element type
template <class T, class M, bool Q8, bool MUL_IR>
Kernel pick(int mode, bool backward) {
  if (backward)
    return mode == kBranch ? backward_kernel<T, M, kBranch, Q8, MUL_IR> : mode == kNorm ? backward_kernel<T, M, kNorm, Q8, MUL_IR> : backward_kernel<T, M, kBoth, Q8, MUL_IR>;
  return mode == kBranch ? forward_kernel<T, M, kBranch, Q8, MUL_IR> : mode == kNorm ? forward_kernel<T, M, kNorm, Q8, MUL_IR> : forward_kernel<T, M, kBoth, Q8, MUL_IR>;
}
template <class T, class M, bool Q8>
Kernel pick(int mode, bool mul_ir, bool backward) { return mul_ir ? pick<T, M, Q8, true>(mode, backward) : pick<T, M, Q8, false>(mode, backward); }
// a file each, so that they compile side by side; _codes: activations in 8 bits
Kernel pick_f32(int mode, bool mul_ir, bool backward);
Kernel pick_f32_codes(int mode, bool mul_ir, bool backward);
Kernel pick_f64(int mode, bool mul_ir, bool backward);
Kernel pick_bf16(int mode, bool mul_ir, bool backward);
Kernel pick_bf16_codes(int mode, bool mul_ir, bool backward);
Kernel pick_f16(int mode, bool mul_ir, bool backward);
Kernel pick_f16_codes(int mode, bool mul_ir, bool backward);

}  // namespace cueq_norm
