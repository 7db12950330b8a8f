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
// What bounds them: HBM.  Every value is read once and written once.  A thread block belongs to one irrep block and a range of
// rows.  It brings the rows' items into shared memory by bulk copies, the next stage while it works on this one; a thread owns
// channels and reads their components there at a stride of dim words (odd: no bank conflicts; neighbouring words in ir_mul),
// so neither layout needs a transposition and sums over components need no other thread.  Results replace the operands in
// shared memory and leave by bulk copies.  A warp, two or four work on one item, by its size (see the plan in norm.cu).
//
// Sums, statistics and all arithmetic are in 32 bits for 16- and 32-bit data, in 64 for 64-bit data; results are rounded once.
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

constexpr int kThreads = 128, kWarps = 4;
constexpr int kMaxBlocks = CUEQ_NORM_MAX_BLOCKS;
enum Mode { kBranch = 1, kNorm = 2, kBoth = 3 };

struct Blk {
  int mul, dim, off, ch;             // off, ch: first element of the block in a row of features, first channel
  int code, gcode, hcode;            // first byte in a row of codes: of y (or x, norm alone), of the gates, of h
  int cta0, ncta, rps, wpi;          // thread blocks, rows per stage, warps per item
  int64_t part;                      // first partial sum
};

struct Params {
  const void *x, *y, *g, *h, *go, *gn;
  int64_t ldx, ldy, ldg, ldh, ldgo, ldgn;
  const void *s, *w;
  void *out, *norm;                  // forward results, rows of `dim_total`
  void *dx, *dy, *dg;
  signed char* codes;
  int64_t ldc;
  void* stats;
  void* parts;
  int64_t parts_len;                 // of one of the two gradients
  int64_t rows;
  double eps;
  int* status;
  int nb, dim_total, channels, ns;   // ns: statistics per (row, block)
  int pdtype, gate, mul_ir, bulk;
  Blk blk[kMaxBlocks];
};

__host__ __device__ constexpr int pad16(int bytes) { return (bytes + 15) & ~15; }

// Byte offsets of a stage's regions.  A region holds one item per row, 16 bytes apart or more.
struct Stage { int a, b, c, d, g, dg, ca, cg, cb, st, total; };

// forward: a = x, b = y, g = gates, ca / cg / cb = codes of y (x), gates, h
__host__ __device__ inline Stage forward_stage(int mode, bool q8, bool gated, int size, int mul, int dim, int rps) {
  Stage s{};
  const int item = pad16(mul * dim * size), gate = pad16(mul * size), code = pad16(mul * dim), gcode = pad16(mul);
  int at = 0;
  auto put = [&](bool on, int bytes) { const int o = at; if (on) at += bytes * rps; return o; };
  s.a = put(true, item);
  s.b = put(mode & kBranch, item);
  s.g = put((mode & kBranch) && gated, gate);
  s.ca = put(q8, code);
  s.cg = put(q8 && (mode & kBranch) && gated, gcode);
  s.cb = put(q8 && mode == kBoth, code);
  s.total = at;
  return s;
}
// backward: a = go, b = gn, c = h, d = y, g = gates, dg = their gradient (over g where that is not in codes), st = statistics
__host__ __device__ inline Stage backward_stage(int mode, bool q8, bool gated, int size, int mul, int dim, int rps, int stat_bytes) {
  Stage s{};
  const int item = pad16(mul * dim * size), gate = pad16(mul * size), code = pad16(mul * dim), gcode = pad16(mul);
  int at = 0;
  auto put = [&](bool on, int bytes) { const int o = at; if (on) at += bytes * rps; return o; };
  s.a = put(mode & kBranch, item);
  s.b = put(mode & kNorm, item);
  s.c = put(mode & kNorm, q8 ? code : item);
  s.d = put(mode & kBranch, q8 ? code : item);
  const bool gates = (mode & kBranch) && gated;
  s.g = put(gates, q8 ? gcode : gate);
  s.dg = q8 ? put(gates, gate) : s.g;
  s.st = put(true, stat_bytes);
  s.total = at;
  return s;
}
// in front of the stages: 2 barriers, room of the reductions, s and w, and (backward) sums of both per group of warps
constexpr int kRed = 16, kRedBytes = 2 * kWarps * 16;
__host__ __device__ inline int head_bytes(int msize, int mul, bool backward, int wpi) {
  return (kRed + kRedBytes + msize * mul * (2 + (backward ? 2 * (kWarps / wpi) : 0)) + 127) & ~127;
}

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

__device__ __forceinline__ float inverse_sqrt(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double inverse_sqrt(double v) { return 1.0 / sqrt(v); }
__device__ __forceinline__ float exponential(float v) { return expf(v); }
__device__ __forceinline__ double exponential(double v) { return exp(v); }
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }   // ordered as |v|, NaN above all
__device__ __forceinline__ unsigned magnitude(double) { return 0u; }                                  // 64-bit data are not kept in codes

template <class M>
__device__ __forceinline__ void activation(int gate, M g, M& v, M& dv) {
  if (gate == CUEQ_NORM_GATE_NONE) { v = M(1); dv = M(0); return; }
  const M e = M(1) / (M(1) + exponential(-g));
  if (gate == CUEQ_NORM_GATE_SIGMOID) { v = e; dv = e * (M(1) - e); }
  else { v = g * e; dv = e * (M(1) + g * (M(1) - e)); }
}

using cueq::code_step;
using cueq::to_code;
__device__ __forceinline__ signed char to_code(double, float) { return 0; }

// ---- a thread block's view of its work --------------------------------------------------------------------------------
template <class M>
struct View {
  M *s, *w, *acc_s, *acc_w;          // parameters and this group's sums, per channel
  unsigned char* red;
  unsigned red_at;
  int mul, dim, su, si;              // strides of a channel and a component inside an item
  int n;                             // values of an item
  int wpi, group, lane, warp_in, tg, gt;   // warps per item; this thread's group, its place in it, the group's threads
  int gate, gated;
  M inv_n, eps;
};

// sum of v and maxima of a, b over the threads that share an item
template <class M>
__device__ __forceinline__ void reduce(View<M>& c, M& v, unsigned& a, unsigned& b) {
  v = cueq::warp_sum(v);
  a = __reduce_max_sync(0xffffffffu, a);
  b = __reduce_max_sync(0xffffffffu, b);
  if (c.wpi == 1) return;
  // two buffers in turn: a thread that writes the third time has passed the second barrier, so all have read the first
  unsigned char* buf = c.red + (c.red_at & 1) * (kWarps * 16);
  ++c.red_at;
  unsigned char* mine = buf + (c.group * c.wpi + c.warp_in) * 16;
  if (c.lane == 0) {
    *reinterpret_cast<M*>(mine) = v;
    reinterpret_cast<unsigned*>(mine)[2] = a;
    reinterpret_cast<unsigned*>(mine)[3] = b;
  }
  if (c.wpi == 4) asm volatile("bar.sync 1, 128;\n" ::: "memory");
  else if (c.group == 0) asm volatile("bar.sync 1, 64;\n" ::: "memory");
  else asm volatile("bar.sync 2, 64;\n" ::: "memory");
  const unsigned char* all = buf + c.group * c.wpi * 16;
  v = M(0);
  for (int k = 0; k < c.wpi; ++k) {
    v += *reinterpret_cast<const M*>(all + k * 16);
    a = max(a, reinterpret_cast<const unsigned*>(all + k * 16)[2]);
    b = max(b, reinterpret_cast<const unsigned*>(all + k * 16)[3]);
  }
}
template <class M>
__device__ __forceinline__ M reduce(View<M>& c, M v) {
  unsigned a = 0, b = 0;
  reduce(c, v, a, b);
  return v;
}

// ---- forward of one item ------------------------------------------------------------------------------------------------
template <class T, class M, int MODE, bool Q8, int DIM>
__device__ __forceinline__ void forward_item(View<M>& c, T* x, T* y, const T* g, signed char* ca, signed char* cg, signed char* cb, M* stats) {
  const int dim = DIM ? DIM : c.dim;
  T* t = (MODE & kBranch) ? y : x;                       // what the first statistic is of
  M sum = M(0);
  unsigned top = 0, gtop = 0;
  for (int u = c.tg; u < c.mul; u += c.gt) {
    const T* p = t + u * c.su;
#pragma unroll
    for (int i = 0; i < dim; ++i) {
      const M v = to<M>(p[i * c.si]);
      sum += v * v;
      if (Q8) top = max(top, magnitude(v));
    }
    if (Q8 && (MODE & kBranch) && c.gated) gtop = max(gtop, magnitude(to<M>(g[u])));
  }
  reduce(c, sum, top, gtop);
  const M r = inverse_sqrt(sum * c.inv_n + c.eps);
  float step = 0.f, inv = 0.f, gstep = 0.f, ginv = 0.f;
  if (Q8) {
    code_step(top, step, inv);
    if ((MODE & kBranch) && c.gated) code_step(gtop, gstep, ginv);
  }
  if (MODE == kNorm) {
    for (int u = c.tg; u < c.mul; u += c.gt) {
      T* p = x + u * c.su;
      const M a = c.w[u] * r;
#pragma unroll
      for (int i = 0; i < dim; ++i) {
        const M v = to<M>(p[i * c.si]);
        if (Q8) ca[u * c.su + i * c.si] = to_code(v, inv);
        p[i * c.si] = from<T>(a * v);
      }
    }
    if (stats && c.tg == 0) { stats[0] = r; stats[2] = M(step); }
    return;
  }
  M hsum = M(0);
  unsigned htop = 0, none = 0;
  for (int u = c.tg; u < c.mul; u += c.gt) {
    M v, dv;
    activation(c.gate, c.gated ? to<M>(g[u]) : M(0), v, dv);
    const M a = c.s[u] * v * r;
    T *px = x + u * c.su, *py = y + u * c.su;
    if (Q8 && c.gated) cg[u] = to_code(to<M>(g[u]), ginv);
#pragma unroll
    for (int i = 0; i < dim; ++i) {
      const M yv = to<M>(py[i * c.si]);
      const M h = to<M>(px[i * c.si]) + a * yv;
      if (Q8) ca[u * c.su + i * c.si] = to_code(yv, inv);
      if (MODE == kBranch) px[i * c.si] = from<T>(h);
      else {
        hsum += h * h;
        if (Q8) htop = max(htop, magnitude(h));
      }
    }
  }
  M rh = M(0);
  float hstep = 0.f, hinv = 0.f;
  if (MODE == kBoth) {
    reduce(c, hsum, htop, none);
    rh = inverse_sqrt(hsum * c.inv_n + c.eps);
    if (Q8) code_step(htop, hstep, hinv);
    // h once more from x and y: kept in 16 bits in between, n would be rounded twice
    for (int u = c.tg; u < c.mul; u += c.gt) {
      M v, dv;
      activation(c.gate, c.gated ? to<M>(g[u]) : M(0), v, dv);
      const M a = c.s[u] * v * r, b = c.w[u] * rh;
      T *px = x + u * c.su, *py = y + u * c.su;
#pragma unroll
      for (int i = 0; i < dim; ++i) {
        const M h = to<M>(px[i * c.si]) + a * to<M>(py[i * c.si]);
        if (Q8) cb[u * c.su + i * c.si] = to_code(h, hinv);
        px[i * c.si] = from<T>(h);
        py[i * c.si] = from<T>(b * h);
      }
    }
  }
  if (stats && c.tg == 0) {
    stats[0] = r; stats[1] = rh; stats[2] = M(step); stats[3] = M(gstep);
    if (Q8 && MODE == kBoth) stats[4] = M(hstep);
  }
}

// ---- backward of one item -----------------------------------------------------------------------------------------------
// go becomes dx behind a branch with a norm, dy behind one without; gn becomes dy or, norm alone, dx; dg the gates' gradient.
// K: type of what was kept (T or codes).
template <class T, class M, class K, int MODE, bool Q8, int DIM>
__device__ __forceinline__ void backward_item(View<M>& c, T* go, T* gn, const K* h, const K* y, const K* g, T* dg, const M* stats, bool has_go) {
  const int dim = DIM ? DIM : c.dim;
  M rh = M(0), qh = M(0);
  if (MODE & kNorm) {
    rh = stats[MODE == kBoth ? 1 : 0];
    const M step = Q8 ? stats[MODE == kBoth ? 4 : 2] : M(1);
    M dot = M(0);
    for (int u = c.tg; u < c.mul; u += c.gt) {
      M p = M(0);
#pragma unroll
      for (int i = 0; i < dim; ++i) p += to<M>(gn[u * c.su + i * c.si]) * to<M>(h[u * c.su + i * c.si]);
      p *= step;
      c.acc_w[u] += rh * p;
      dot += c.w[u] * p;
    }
    dot = reduce(c, dot);
    qh = rh * (rh * c.inv_n * dot) * step;
    if (MODE == kNorm) {
      for (int u = c.tg; u < c.mul; u += c.gt) {
        const M a = c.w[u];
#pragma unroll
        for (int i = 0; i < dim; ++i) {
          const int e = u * c.su + i * c.si;
          gn[e] = from<T>(rh * (a * to<M>(gn[e]) - qh * to<M>(h[e])));
        }
      }
      return;
    }
  }
  const M r = stats[0];
  const M step = Q8 ? stats[2] : M(1), gstep = Q8 ? stats[3] : M(1);
  M dot = M(0);
  for (int u = c.tg; u < c.mul; u += c.gt) {
    M v, dv, p = M(0);
    activation(c.gate, c.gated ? to<M>(g[u]) * gstep : M(0), v, dv);
    const M b = MODE == kBoth ? c.w[u] : M(0);
#pragma unroll
    for (int i = 0; i < dim; ++i) {
      const int e = u * c.su + i * c.si;
      M o = MODE == kBranch || has_go ? to<M>(go[e]) : M(0);
      if (MODE == kBoth) o += rh * (b * to<M>(gn[e]) - qh * to<M>(h[e]));
      p += o * to<M>(y[e]);
    }
    p *= step;
    const M s = c.s[u];
    c.acc_s[u] += v * r * p;
    dot += s * v * p;
    if (c.gated && !Q8) continue;                        // g is read once more below, before dg replaces it
    if (c.gated) dg[u] = from<T>(s * dv * r * p);
  }
  dot = reduce(c, dot);
  const M q = r * (r * c.inv_n * dot) * step;
  for (int u = c.tg; u < c.mul; u += c.gt) {
    M v, dv, p = M(0);
    activation(c.gate, c.gated ? to<M>(g[u]) * gstep : M(0), v, dv);
    const M a = c.s[u] * v, b = MODE == kBoth ? c.w[u] : M(0);
#pragma unroll
    for (int i = 0; i < dim; ++i) {
      const int e = u * c.su + i * c.si;
      M o = MODE == kBranch || has_go ? to<M>(go[e]) : M(0);
      if (MODE == kBoth) o += rh * (b * to<M>(gn[e]) - qh * to<M>(h[e]));
      const M yv = to<M>(y[e]);
      if (!Q8) p += o * yv;
      const T dy = from<T>(r * (a * o - q * yv));
      if (MODE == kBoth) { go[e] = from<T>(o); gn[e] = dy; } else go[e] = dy;
    }
    if (c.gated && !Q8) dg[u] = from<T>(c.s[u] * dv * r * p);
  }
}

// ---- moving items -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void bulk_in(void* dst, const void* src, unsigned bytes, unsigned long long* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
               ::"r"(s32(dst)), "l"(src), "r"(bytes), "r"(s32(bar)) : "memory");
}
__device__ __forceinline__ void bulk_out(void* dst, const void* src, unsigned bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(dst), "r"(s32(src)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;\n" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory"); }

// A region of a stage and the rows in memory that it holds: `size` bytes an element (1: codes).
struct Move { int region, pitch, bytes, size; const unsigned char* src; unsigned char* dst; int64_t ld; };

// Rows [z0, z0 + n) of every region, plain: consecutive threads take consecutive elements.
__device__ __forceinline__ void copy_rows(const Move& m, unsigned char* stage, int64_t z0, int n, bool in) {
  for (int r = 0; r < n; ++r) {
    unsigned char* a = stage + m.region + r * m.pitch;
    if (in) {
      const unsigned char* b = m.src + (z0 + r) * m.ld;
      if (m.size == 2) for (int e = threadIdx.x; e < m.bytes / 2; e += kThreads) reinterpret_cast<unsigned short*>(a)[e] = __ldg(reinterpret_cast<const unsigned short*>(b) + e);
      else if (m.size == 4) for (int e = threadIdx.x; e < m.bytes / 4; e += kThreads) reinterpret_cast<unsigned*>(a)[e] = __ldg(reinterpret_cast<const unsigned*>(b) + e);
      else if (m.size == 8) for (int e = threadIdx.x; e < m.bytes / 8; e += kThreads) reinterpret_cast<unsigned long long*>(a)[e] = __ldg(reinterpret_cast<const unsigned long long*>(b) + e);
      else for (int e = threadIdx.x; e < m.bytes / 16; e += kThreads) reinterpret_cast<uint4*>(a)[e] = __ldg(reinterpret_cast<const uint4*>(b) + e);
    } else {
      unsigned char* b = m.dst + (z0 + r) * m.ld;
      if (m.size == 2) for (int e = threadIdx.x; e < m.bytes / 2; e += kThreads) reinterpret_cast<unsigned short*>(b)[e] = reinterpret_cast<unsigned short*>(a)[e];
      else if (m.size == 4) for (int e = threadIdx.x; e < m.bytes / 4; e += kThreads) reinterpret_cast<unsigned*>(b)[e] = reinterpret_cast<unsigned*>(a)[e];
      else if (m.size == 8) for (int e = threadIdx.x; e < m.bytes / 8; e += kThreads) reinterpret_cast<unsigned long long*>(b)[e] = reinterpret_cast<unsigned long long*>(a)[e];
      else for (int e = threadIdx.x; e < m.bytes / 16; e += kThreads) reinterpret_cast<uint4*>(b)[e] = reinterpret_cast<uint4*>(a)[e];
    }
  }
}

// Rows first .. last in stages of rps rows: loads, work on a stage, stores.  Loads and stores of row r of a stage are issued by
// lane r of warp 0, so that a lane's own wait for its stores' reads covers the memory that its next loads overwrite.
template <int NIN, int NOUT, class Work>
__device__ __forceinline__ void run_stages(const Params& p, const Blk& b, int64_t first, int64_t last, const Move (&in)[NIN], int nin,
                                           const Move (&out)[NOUT], int nout, unsigned char* stages, int stage_bytes, unsigned long long* full,
                                           Work work) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (!p.bulk) {
    for (int64_t z = first; z < last; z += b.rps) {
      const int n = (int)min((int64_t)b.rps, last - z);
#pragma unroll
      for (int k = 0; k < NIN; ++k) if (k < nin) copy_rows(in[k], stages, z, n, true);
      __syncthreads();
      work(stages, z, n);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NOUT; ++k) if (k < nout) copy_rows(out[k], stages, z, n, false);
      __syncthreads();
    }
    return;
  }
  unsigned row_bytes = 0;
#pragma unroll
  for (int k = 0; k < NIN; ++k) if (k < nin) row_bytes += in[k].bytes;
  auto load = [&](int64_t z, int s) {
    const int n = (int)min((int64_t)b.rps, last - z);
    if (lane == 0) bar_expect_tx(full + s, n * row_bytes);
    __syncwarp();
    if (lane < n) {
#pragma unroll
      for (int k = 0; k < NIN; ++k)
        if (k < nin) bulk_in(stages + s * stage_bytes + in[k].region + lane * in[k].pitch, in[k].src + (z + lane) * in[k].ld, in[k].bytes, full + s);
    }
  };
  if (warp == 0 && first < last) load(first, 0);
  unsigned it = 0;
  for (int64_t z = first; z < last; z += b.rps, ++it) {
    const int s = it & 1, n = (int)min((int64_t)b.rps, last - z);
    const bool more = z + b.rps < last;
    if (warp == 0 && more) {
      bulk_wait_read();                                  // this lane's stores from the other stage
      load(z + b.rps, s ^ 1);
    }
    const bool ok = bar_wait(full + s, (it >> 1) & 1, p.status);
    if (!__syncthreads_and(ok)) {                        // a copy did not arrive in time: give up once the copies in flight have landed
      if (more) bar_wait(full + (s ^ 1), ((it + 1) >> 1) & 1, p.status);
      bar_wait(full + s, (it >> 1) & 1, p.status);
      break;
    }
    work(stages + s * stage_bytes, z, n);
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    __syncthreads();
    if (warp == 0) {
      if (lane < n) {
#pragma unroll
        for (int k = 0; k < NOUT; ++k)
          if (k < nout) bulk_out(out[k].dst + (z + lane) * out[k].ld, stages + s * stage_bytes + out[k].region + lane * out[k].pitch, out[k].bytes);
      }
      bulk_commit();
    }
  }
  if (warp == 0) bulk_wait_read();
}

template <class M>
__device__ __forceinline__ View<M> make_view(const Params& p, const Blk& b, unsigned char* smem, bool backward) {
  View<M> c;
  c.mul = b.mul; c.dim = b.dim; c.n = b.mul * b.dim;
  c.su = p.mul_ir ? b.dim : 1;
  c.si = p.mul_ir ? 1 : b.mul;
  c.wpi = b.wpi;
  const int warp = threadIdx.x >> 5;
  c.lane = threadIdx.x & 31;
  c.group = warp / b.wpi;
  c.warp_in = warp % b.wpi;
  c.tg = c.warp_in * 32 + c.lane;
  c.gt = b.wpi * 32;
  c.gate = p.gate; c.gated = p.gate != CUEQ_NORM_GATE_NONE;
  c.inv_n = M(1) / M(c.n);
  c.eps = M(p.eps);
  c.red = smem + kRed;
  c.red_at = 0;
  c.s = reinterpret_cast<M*>(smem + kRed + kRedBytes);
  c.w = c.s + b.mul;
  c.acc_s = c.w + b.mul + c.group * b.mul;
  c.acc_w = c.w + b.mul + (kWarps / b.wpi + c.group) * b.mul;
  for (int u = threadIdx.x; u < b.mul; u += kThreads) {
    c.s[u] = p.s ? cueq::load_as<M>(p.s, p.pdtype, b.ch + u) : M(1);
    c.w[u] = p.w ? cueq::load_as<M>(p.w, p.pdtype, b.ch + u) : M(1);
  }
  if (backward)
    for (int u = threadIdx.x; u < 2 * (kWarps / b.wpi) * b.mul; u += kThreads) c.w[b.mul + u] = M(0);
  if (threadIdx.x == 0) {
    bar_init(reinterpret_cast<unsigned long long*>(smem), 1);
    bar_init(reinterpret_cast<unsigned long long*>(smem) + 1, 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  return c;
}

__device__ __forceinline__ const Blk& my_block(const Params& p) {
  int k = 0;
  while (k + 1 < p.nb && (int)blockIdx.x >= p.blk[k + 1].cta0) ++k;
  return p.blk[k];
}

#define CUEQ_NORM_DIMS(dim, CALL)      \
  switch (dim) {                       \
    case 1: { CALL(1); break; }        \
    case 3: { CALL(3); break; }        \
    case 5: { CALL(5); break; }        \
    case 7: { CALL(7); break; }        \
    default: { CALL(0); break; }       \
  }

template <class T, class M, int MODE, bool Q8>
__global__ void __launch_bounds__(kThreads, sizeof(M) == 8 ? 4 : 8) forward_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  const Blk& b = my_block(p);
  View<M> c = make_view<M>(p, b, smem, false);
  const int j = blockIdx.x - b.cta0, size = sizeof(T);
  const int64_t first = p.rows * j / b.ncta, last = p.rows * (j + 1) / b.ncta;
  const Stage st = forward_stage(MODE, Q8, c.gated, size, b.mul, b.dim, b.rps);
  const int item = b.mul * b.dim * size, gate = b.mul * size, code = pad16(b.mul * b.dim), gcode = pad16(b.mul);
  const bool branch = MODE & kBranch;
  auto at = [](const void* q, int64_t bytes) { return reinterpret_cast<unsigned char*>(const_cast<void*>(q)) + bytes; };
  const int64_t ldo = (int64_t)p.dim_total * size;
  const Move in[3] = {{st.a, pad16(item), item, size, at(p.x, (int64_t)b.off * size), nullptr, p.ldx * size},
                      {st.b, pad16(item), item, size, at(p.y, (int64_t)b.off * size), nullptr, p.ldy * size},
                      {st.g, pad16(gate), gate, size, at(p.g, (int64_t)b.ch * size), nullptr, p.ldg * size}};
  const Move o_out = {st.a, pad16(item), item, size, nullptr, at(branch ? p.out : p.norm, (int64_t)b.off * size), ldo};
  const Move o_norm = {st.b, pad16(item), item, size, nullptr, at(p.norm, (int64_t)b.off * size), ldo};
  const Move o_ca = {st.ca, code, code, 16, nullptr, (unsigned char*)p.codes + b.code, p.ldc};
  const Move o_cg = {st.cg, gcode, gcode, 16, nullptr, (unsigned char*)p.codes + b.gcode, p.ldc};
  const Move o_cb = {st.cb, code, code, 16, nullptr, (unsigned char*)p.codes + b.hcode, p.ldc};
  // results in an order in which those that a call does not have come last
  const Move out[5] = {o_out, MODE == kBoth ? o_norm : o_ca, MODE == kBoth ? o_ca : o_cg, MODE == kBoth ? o_cb : o_cg, o_cg};
  const int nout = 1 + (MODE == kBoth) + (Q8 ? 1 + (MODE == kBoth) + (branch && c.gated) : 0);
  const int k = (int)(&b - p.blk);
  run_stages(p, b, first, last, in, branch ? 2 + c.gated : 1, out, nout, smem + head_bytes(sizeof(M), b.mul, false, b.wpi), st.total,
             reinterpret_cast<unsigned long long*>(smem), [&](unsigned char* s, int64_t z, int n) {
    for (int r = c.group; r < n; r += kWarps / c.wpi) {
      M* stats = p.stats ? reinterpret_cast<M*>(p.stats) + ((z + r) * p.nb + k) * p.ns : nullptr;
#define CUEQ_CALL(D)                                                                                                              \
  forward_item<T, M, MODE, Q8, D>(c, reinterpret_cast<T*>(s + st.a + r * pad16(item)), reinterpret_cast<T*>(s + st.b + r * pad16(item)), \
                                  reinterpret_cast<const T*>(s + st.g + r * pad16(gate)), reinterpret_cast<signed char*>(s + st.ca + r * code), \
                                  reinterpret_cast<signed char*>(s + st.cg + r * gcode), reinterpret_cast<signed char*>(s + st.cb + r * code), stats)
      CUEQ_NORM_DIMS(b.dim, CUEQ_CALL)
#undef CUEQ_CALL
    }
  });
}

template <class T, bool Q8> struct Kept { using type = T; };
template <class T> struct Kept<T, true> { using type = signed char; };

template <class T, class M, int MODE, bool Q8>
__global__ void __launch_bounds__(kThreads, sizeof(M) == 8 ? 4 : 8) backward_kernel(const __grid_constant__ Params p) {
  using K = typename Kept<T, Q8>::type;
  extern __shared__ __align__(128) unsigned char smem[];
  const Blk& b = my_block(p);
  View<M> c = make_view<M>(p, b, smem, true);
  const int j = blockIdx.x - b.cta0, size = sizeof(T);
  const int64_t first = p.rows * j / b.ncta, last = p.rows * (j + 1) / b.ncta;
  const int stat = p.ns * (int)sizeof(M);
  const Stage st = backward_stage(MODE, Q8, c.gated, size, b.mul, b.dim, b.rps, stat);
  const int item = b.mul * b.dim * size, gate = b.mul * size, code = pad16(b.mul * b.dim), gcode = pad16(b.mul);
  const bool branch = MODE & kBranch, has_go = p.go != nullptr;
  auto at = [](const void* q, int64_t bytes) { return reinterpret_cast<unsigned char*>(const_cast<void*>(q)) + bytes; };
  const int64_t fo = (int64_t)b.off * size, go_ = (int64_t)b.ch * size, ldo = (int64_t)p.dim_total * size;
  const int kpitch = Q8 ? code : pad16(item), kbytes = Q8 ? code : item, ksize = Q8 ? 16 : size;
  const int k = (int)(&b - p.blk);
  const Move i_go = {st.a, pad16(item), item, size, at(p.go, fo), nullptr, p.ldgo * size};
  const Move i_gn = {st.b, pad16(item), item, size, at(p.gn, fo), nullptr, p.ldgn * size};
  const Move i_h = {st.c, kpitch, kbytes, ksize, Q8 ? (unsigned char*)p.codes + (MODE == kBoth ? b.hcode : b.code) : at(p.h, fo), nullptr,
                    Q8 ? p.ldc : p.ldh * size};
  const Move i_y = {st.d, kpitch, kbytes, ksize, Q8 ? (unsigned char*)p.codes + b.code : at(p.y, fo), nullptr, Q8 ? p.ldc : p.ldy * size};
  const Move i_g = {st.g, Q8 ? gcode : pad16(gate), Q8 ? gcode : gate, Q8 ? 16 : size, Q8 ? (unsigned char*)p.codes + b.gcode : at(p.g, go_),
                    nullptr, Q8 ? p.ldc : p.ldg * size};
  const Move i_st = {st.st, stat, stat, 16, (unsigned char*)p.stats + (int64_t)k * stat, nullptr, (int64_t)p.nb * stat};
  // operands in an order in which those that a call does not have come last
  const Move in[6] = {i_st, branch ? i_y : i_h, branch ? (MODE == kBoth ? i_h : i_go) : i_gn, MODE == kBoth ? i_gn : i_g,
                      MODE == kBoth && c.gated ? i_g : i_go, i_go};
  const int nin = MODE == kNorm ? 3 : MODE == kBranch ? 3 + c.gated : 4 + c.gated + has_go;
  const Move o_a = {st.a, pad16(item), item, size, nullptr, at(branch && MODE == kBoth ? p.dx : p.dy, fo), ldo};
  const Move o_b = {st.b, pad16(item), item, size, nullptr, at(branch ? p.dy : p.dx, fo), ldo};
  const Move o_g = {st.dg, pad16(gate), gate, size, nullptr, at(p.dg, go_), (int64_t)p.channels * size};
  const Move out[3] = {MODE == kNorm ? o_b : o_a, MODE == kBoth ? o_b : o_g, o_g};
  const int nout = MODE == kNorm ? 1 : 1 + (MODE == kBoth) + c.gated;
  run_stages(p, b, first, last, in, nin, out, nout, smem + head_bytes(sizeof(M), b.mul, true, b.wpi), st.total,
             reinterpret_cast<unsigned long long*>(smem), [&](unsigned char* s, int64_t, int n) {
    for (int r = c.group; r < n; r += kWarps / c.wpi) {
#define CUEQ_CALL(D)                                                                                                              \
  backward_item<T, M, K, MODE, Q8, D>(c, reinterpret_cast<T*>(s + st.a + r * pad16(item)), reinterpret_cast<T*>(s + st.b + r * pad16(item)), \
                                      reinterpret_cast<const K*>(s + st.c + r * kpitch), reinterpret_cast<const K*>(s + st.d + r * kpitch),  \
                                      reinterpret_cast<const K*>(s + st.g + r * (Q8 ? gcode : pad16(gate))),                      \
                                      reinterpret_cast<T*>(s + st.dg + r * pad16(gate)), reinterpret_cast<const M*>(s + st.st + r * stat), has_go)
      CUEQ_NORM_DIMS(b.dim, CUEQ_CALL)
#undef CUEQ_CALL
    }
  });
  // this thread block's sums of the parameters' gradients, its groups in order
  __syncthreads();
  const int ng = kWarps / b.wpi;
  for (int u = threadIdx.x; u < b.mul; u += kThreads) {
    M vs = M(0), vw = M(0);
    for (int k2 = 0; k2 < ng; ++k2) { vs += c.w[b.mul + k2 * b.mul + u]; vw += c.w[b.mul + (ng + k2) * b.mul + u]; }
    M* dst = reinterpret_cast<M*>(p.parts) + b.part + (int64_t)j * b.mul + u;
    if (MODE & kBranch) dst[0] = vs;
    if (MODE & kNorm) dst[p.parts_len] = vw;
  }
}

using Kernel = void (*)(Params);

// the kernels of one element type, [mode - 1][q8]
template <class T, class M, bool Q8>
Kernel pick(int mode, bool backward) {
  if (backward)
    return mode == kBranch ? backward_kernel<T, M, kBranch, Q8> : mode == kNorm ? backward_kernel<T, M, kNorm, Q8> : backward_kernel<T, M, kBoth, Q8>;
  return mode == kBranch ? forward_kernel<T, M, kBranch, Q8> : mode == kNorm ? forward_kernel<T, M, kNorm, Q8> : forward_kernel<T, M, kBoth, Q8>;
}
Kernel pick_f32(int mode, bool q8, bool backward);
Kernel pick_f64(int mode, bool q8, bool backward);
Kernel pick_bf16(int mode, bool q8, bool backward);
Kernel pick_f16(int mode, bool q8, bool backward);

}  // namespace cueq_norm
