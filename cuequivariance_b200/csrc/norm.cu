// Host side of the norm kernels (norm_kernels.cuh): argument checks, the division of rows and irrep blocks among thread blocks,
// and the sum over thread blocks of the parameters' gradients.
#include <cstring>

#include "norm_kernels.cuh"

namespace {

using namespace cueq_norm;

constexpr int kSmemPerSm = 227 * 1024;
constexpr int kSliceValues = 1024;       // neighbouring irrep blocks are put together up to this length
constexpr int kWarpsOfLongBlocks = 9, kFewWarps = 7;
constexpr int kStageBytes = 4096;        // rows are put together up to about this much per stage

int element_size(int dtype) { return dtype == CUEQ_F64 ? 8 : dtype == CUEQ_F32 ? 4 : 2; }
bool gated(const cueq_norm_args* a) { return a->gate != CUEQ_NORM_GATE_NONE && (a->mode & kBranch); }
// the backward pass forms h again from x (kAgain)
bool again(const cueq_norm_args* a) { return a->mode == kBoth && !a->codes && element_size(a->dtype) == 2; }
// a branch whose norm has no cotangent is differentiated alone, with the statistics that both have left
int stats_per_item(const cueq_norm_args* a) { return a->stats_stride ? a->stats_stride : a->codes && a->mode == kBoth ? 8 : 4; }

int check(const cueq_norm_args* a) {
  if (!a) return cueq::fail("norm: null arguments");
  if (a->struct_bytes != (int)sizeof(cueq_norm_args)) return cueq::fail("norm: the binding declares another argument block");
  if (a->mode < CUEQ_NORM_BRANCH || a->mode > CUEQ_NORM_BOTH) return cueq::fail("norm: unknown mode %d", a->mode);
  if (a->gate < CUEQ_NORM_GATE_NONE || a->gate > CUEQ_NORM_GATE_SILU) return cueq::fail("norm: unknown gate %d", a->gate);
  if (a->dtype < CUEQ_F32 || a->dtype > CUEQ_F16 || a->param_dtype < CUEQ_F32 || a->param_dtype > CUEQ_F16) return cueq::fail("norm: unknown element type");
  if (a->num_blocks < 1 || a->num_blocks > kMaxBlocks || !a->blocks) return cueq::fail("norm: between 1 and %d irrep blocks", kMaxBlocks);
  if (a->rows < 0 || a->rows >= (int64_t(1) << 40)) return cueq::fail("norm: bad number of rows");
  for (int k = 0; k < a->num_blocks; ++k)
    if (a->blocks[k].mul < 1 || a->blocks[k].dim < 1 || a->blocks[k].dim > 32767 || (int64_t)a->blocks[k].mul * a->blocks[k].dim > (1 << 20)) return cueq::fail("norm: bad irrep block %d", k);
  if (a->stats_stride && a->stats_stride != 8 && (a->stats_stride != 4 || (a->codes && a->mode == kBoth))) return cueq::fail("norm: bad stride of the statistics");
  // in 32 bits eps has to be a normal number: an empty block is multiplied by eps^-1/2
  if (!(a->eps > 0) || a->eps > 1e300 || (a->dtype != CUEQ_F64 && ((float)a->eps < 1.17549435e-38f || a->eps > 1e38)))
    return cueq::fail("norm: eps must be positive, finite and, but for 64-bit data, a normal 32-bit number");
  if (a->codes && a->dtype == CUEQ_F64) return cueq::fail("norm: 64-bit data are not kept in 8 bits");
  return 0;
}

// bytes of a row of codes: y (or x) block by block, the gates, out; every block from a 16-byte boundary on
int64_t code_layout(const cueq_norm_args* a, Params* p) {
  int64_t at = 0;
  for (int k = 0; k < a->num_blocks; ++k) { if (p) p->blk[k].code = (int)at; at += pad16(a->blocks[k].mul * a->blocks[k].dim); }
  if (gated(a)) for (int k = 0; k < a->num_blocks; ++k) { if (p) p->blk[k].gcode = (int)at; at += pad16(a->blocks[k].mul); }
  if (a->mode == kBoth) for (int k = 0; k < a->num_blocks; ++k) { if (p) p->blk[k].hcode = (int)at; at += pad16(a->blocks[k].mul * a->blocks[k].dim); }
  return at;
}

enum { kTooLong = 1, kTooLongForUnits = 2 };

// Which way each tensor moves, for slices that are `whole` rows or parts of rows that start and end on 16-byte boundaries (`even`).
void set_routes(const cueq_norm_args* a, bool backward, Params* p, bool whole, bool even) {
  const int size = element_size(a->dtype);
  auto route = [&](const void* q, int64_t ld, int64_t width) -> signed char {
    if (((uintptr_t)q & 15) || (!even && !whole)) return kPlain;
    if (whole && ld == width) return kDense;
    return even && ld * size % 16 == 0 ? kRows : kPlain;
  };
  const int64_t d = p->dim_total, c = p->channels;
  p->route[tX] = route(a->x, a->ldx, d); p->route[tY] = route(a->y, a->ldy, d); p->route[tH] = again(a) ? p->route[tX] : route(a->h, a->ldh, d);
  p->route[tGo] = route(a->go, a->ldgo, d); p->route[tGn] = route(a->gn, a->ldgn, d); p->route[tG] = route(a->g, a->ldg, c);
  p->route[tOut] = route(a->out, d, d); p->route[tNorm] = route(a->norm, d, d);
  p->route[tDx] = route(a->dx, d, d); p->route[tDy] = route(a->dy, d, d); p->route[tDg] = route(a->dg, c, c);
  p->route[tStats] = whole ? kDense : kRows;
  // An operand and the result in its place have rows at one distance: dense together, or each row by itself where that is possible.
  auto pair = [&](int in, int out) {
    if ((p->route[in] == kDense) == (p->route[out] == kDense)) return;
    const int t = p->route[in] == kDense ? in : out;
    p->route[t] = even ? kRows : kPlain;
  };
  if (!backward) {
    pair(tX, a->mode & kBranch ? tOut : tNorm);
    if (a->mode == kBoth) pair(tY, tNorm);
  } else {
    if (a->mode == kBranch) pair(tGo, tDy);
    if (a->mode == kNorm) pair(tGn, tDx);
    if (a->mode == kBoth) { if (a->go) pair(tGo, tDx); pair(tGn, tDy); }
    if (gated(a) && !a->codes) pair(tG, tDg);
  }
}

// Lanes that issue the copies of a stage of rps rows, in or out (the larger).
int copy_lanes(const cueq_norm_args* a, bool backward, const Params& p, int rps) {
  const bool branch = a->mode & kBranch, norm = a->mode & kNorm, gate = gated(a), q8 = a->codes != nullptr, both = a->mode == kBoth;
  auto lanes = [&](bool on, int t) { return !on || p.route[t] == kPlain ? 0 : p.route[t] == kDense ? 1 : rps; };
  const int codes = q8 ? (1 + both + gate) * rps : 0;
  int in, out;
  if (!backward) {
    in = lanes(true, tX) + lanes(branch, tY) + lanes(gate, tG);
    out = lanes(branch, tOut) + lanes(norm, tNorm) + codes;
  } else {
    in = lanes(true, tStats) + lanes(branch && a->go, tGo) + lanes(norm, tGn) + (q8 ? codes : lanes(norm, tH) + lanes(branch, tY) + lanes(gate, tG));
    out = lanes(norm, tDx) + lanes(branch, tDy) + lanes(gate, tDg);
  }
  return in > out ? in : out;
}

// Divides the work: neighbouring irrep blocks to slices of at most kSliceValues values (a longer block is a slice by itself); the warps that
// shared memory and registers hold at a time share the rows of every slice.  (Warps of one slice each, in proportion to its length,
// were 35 % idle in the end: no length says what a slice costs.)  Rows that are dense but no multiple of 16 bytes come in stages of 2, 4 or 8, which are.
int make_plan(const cueq_norm_args* a, bool backward, bool dense, Params* p, int* grid, int* smem_bytes) {
  const bool q8 = a->codes != nullptr, gate = gated(a);
  const int size = element_size(a->dtype), msize = a->dtype == CUEQ_F64 ? 8 : 4, stat = p->ns * msize;
  int ns = 0;
  bool even = true;
  // A slice that starts off a 16-byte boundary, or rows that do, would move element by element: as long as one fits, a longer slice that does not is
  // better (13x0e+57x1o+9x2e+201x3o, 20,510 rows in float32, gated residual: 373 + 449 us in two slices, 127 + 135 in one).
  int64_t width = 0, gates = 0;
  for (int k = 0; k < a->num_blocks; ++k) { width += (int64_t)a->blocks[k].mul * a->blocks[k].dim; gates += a->blocks[k].mul; }
  const bool aligned_rows = width * size % 16 == 0 && (!gate || gates * size % 16 == 0);
  for (int k = 0; k < a->num_blocks; ++k) {
    Blk& b = p->blk[k];
    b.mul = a->blocks[k].mul; b.dim = (short)a->blocks[k].dim;
    b.off = p->dim_total; b.ch = p->channels;
    const int n = b.mul * b.dim;
    const bool may_start = !dense || (aligned_rows && b.off * size % 16 == 0 && (!gate || b.ch * size % 16 == 0));
    if (!ns || (p->slice[ns - 1].values + n > kSliceValues && may_start)) { p->slice[ns] = Slice{}; p->slice[ns].first = (short)k; ++ns; }
    Slice& s = p->slice[ns - 1];
    if (s.count == 0 && (b.off * size % 16 || (gated(a) && b.ch * size % 16))) even = false;
    ++s.count; s.values += n; s.channels += b.mul;
    p->dim_total += n; p->channels += b.mul;
  }
  if (p->dim_total * size % 16 || (gated(a) && p->channels * size % 16)) even = false;
  p->num_slices = ns; p->nb = a->num_blocks;
  // sizes from here on stay below a few MB: every pass has a row of a slice's values in shared memory
  for (int k = 0; k < ns; ++k)
    if ((int64_t)p->slice[k].values * size > kSmemPerSm) return dense && p->slice[k].count > 1 ? kTooLongForUnits : kTooLong;
  set_routes(a, backward, p, dense && ns == 1, even);
  int unit = 1;                                          // rows after which dense rows are on a 16-byte boundary again
  if (dense && ns == 1) while (unit < 8 && (unit * p->dim_total * size % 16 || (gated(a) && unit * p->channels * size % 16))) unit *= 2;
  auto stage = [&](const Slice& s) { return backward ? backward_stage(*p, s, a->mode, q8, size, stat).total : forward_stage(*p, s, a->mode, q8, size).total; };
  auto need = [&](const Slice& s, int stages) { return head_bytes(msize, s, a->mode, backward) + stages * stage(s); };
  // How a block is worked on: up to 32, 64 or 128 channels by 1, 2 or 4 per lane, where these are neighbours on a boundary of as many
  // values in every row; up to 16 channels with several rows side by side.  The rest, l > 3 among it, goes through loops (256 channels: 0.6
  // of the copy bandwidth where 128 have 0.75).
  for (int q = 0; q < ns; ++q) {
    Slice& s = p->slice[q];
    const Blk& b0 = p->blk[s.first];
    for (int k = s.first; k < s.first + s.count; ++k) {
      Blk& b = p->blk[k];
      const int per = b.mul <= 32 ? 1 : b.mul <= 64 ? 2 : 4;
      const int places = (b.off - b0.off) | (b.ch - b0.ch) | b.mul | s.values | s.channels;
      b.per_lane = b.dim <= 7 && b.dim % 2 && b.mul <= 128 && places % per == 0 ? per : 0;
      b.lanes = 32;
      while (b.per_lane == 1 && b.lanes / 2 >= b.mul) b.lanes /= 2;
      b.sum = s.sums;
      s.sums += pad4(b.lanes < 32 ? 32 : b.mul);
      if (!b.per_lane) s.loops = 1;
    }
  }
  p->unit = unit;
  int smem = 0;
  for (int k = 0; k < ns; ++k) {
    Slice& s = p->slice[k];
    s.rps = (short)unit;
    if (dense && s.values > kSliceValues && s.count > 1 && need(s, 1) > kSmemPerSm / 3) return kTooLongForUnits;
    if (unit > 1 && need(s, 1) > kSmemPerSm / 3) return kTooLongForUnits;
    const int one = stage(s) / unit;
    int rps = kStageBytes / (one ? one : 1) / unit * unit, beside = 1;
    for (int k2 = s.first; k2 < s.first + s.count; ++k2) beside = 32 / p->blk[k2].lanes > beside ? 32 / p->blk[k2].lanes : beside;
    while (rps < beside && (rps + unit) * one <= 2 * kStageBytes) rps += unit;   // rows that a warp takes side by side
    rps = rps >= 3 ? (rps + 1) / 4 * 4 : rps;            // rows are worked on by fours, twos or one by one
    s.rps = (short)(rps < unit ? unit : rps > 32 ? 32 : rps);
    while (s.rps > unit && copy_lanes(a, backward, *p, s.rps) > 32) s.rps -= unit;
  }
  auto fit = [&](int stages) {                           // warps per SM, 0: none
    p->stages = stages;
    smem = 0;
    for (int k = 0; k < ns; ++k) { const int b = need(p->slice[k], stages); smem = b > smem ? b : smem; }
    *smem_bytes = smem;
    return smem > kSmemPerSm ? 0 : smem + 1024 > kSmemPerSm ? 1 : kSmemPerSm / (smem + 1024);
  };
  // Where two stages leave room for few warps, twice as many with one stage each are better (256x(0e+1o+2e+3o) with the next norm, backward:
  // 348 us with four warps, 239 with eight).
  int occupancy = fit(2);
  if (occupancy < kFewWarps) occupancy = fit(1);
  if (occupancy < 1) return kTooLong;
  occupancy = occupancy > warps_per_sm(msize) ? warps_per_sm(msize) : occupancy;
  // Long blocks in full are bound by HBM, which serves 9 warps per SM with 60 KB under way better than 14 (32,768 rows of 128x(0e+1o+2e+3o) in
  // float32: norm 155 and 168 us backward, gated residual 155 and 164 us forward); the others are bound by instructions and want all
  // (64x0e, gated residual: 123 us, with 8 warps 167 us).
  if (a->mode != kBoth && !q8 && size >= 4 && p->dim_total / a->num_blocks >= 384 && occupancy > kWarpsOfLongBlocks) occupancy = kWarpsOfLongBlocks;
  const int64_t units = (a->rows + unit - 1) / unit * ns, warps = (int64_t)kSms * occupancy;
  *grid = (int)(units < warps ? units : warps);
  if (*grid) { p->deal = units / *grid; p->deal_more = (int)(units % *grid); }
  return 0;
}

int fill(const cueq_norm_args* a, bool backward, Params* p, int* grid, int* smem) {
  if (int rc = check(a)) return rc;
  int rc = kTooLongForUnits;
  for (int dense = 1; dense >= 0 && rc == kTooLongForUnits; --dense) {
    std::memset(p, 0, sizeof(*p));
    p->ns = stats_per_item(a);
    p->gate = a->mode & kBranch ? a->gate : CUEQ_NORM_GATE_NONE;
    p->go = a->go;
    code_layout(a, p);
    rc = make_plan(a, backward, dense, p, grid, smem);
  }
  if (rc) return cueq::fail("norm: a row of an irrep block does not fit into shared memory (%d bytes)", kSmemPerSm);
  return 0;
}

// dscale, dweight: the warps' sums of a channel, in order
struct SumParams {
  const void* parts;
  void* out[2];
  int warps, channels, dtype;
  const int* status;
};
constexpr int kSumRows = 128, kSumChannels = 8;   // eight channels, a sector of a warp's sums; 1,800 warps in 14 steps (32 x 32 threads: 50 steps, 8 us)
template <class M>
__global__ void __launch_bounds__(kSumChannels * kSumRows) sum_kernel(const __grid_constant__ SumParams p) {
  __shared__ M partial[kSumRows][kSumChannels + 1];
  if (!cueq_tc::status_clean(p.status)) return;           // a warp that gave up has left no sums
  const int ch = blockIdx.x * kSumChannels + threadIdx.x;
  const int which = blockIdx.y;
  M v = M(0);
  if (ch < p.channels && p.out[which]) {
    const M* src = reinterpret_cast<const M*>(p.parts) + (int64_t)which * p.warps * p.channels + ch;
#pragma unroll 8
    for (int j = threadIdx.y; j < p.warps; j += kSumRows) v += src[(int64_t)j * p.channels];
  }
  partial[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
#pragma unroll
  for (int n = kSumRows / 2; n >= 4; n /= 2) {
    if (threadIdx.y < n) partial[threadIdx.y][threadIdx.x] += partial[threadIdx.y + n][threadIdx.x];
    __syncthreads();
  }
  if (threadIdx.y || ch >= p.channels || !p.out[which]) return;
  v = M(0);
#pragma unroll
  for (int j = 0; j < 4; ++j) v += partial[j][threadIdx.x];
  switch (p.dtype) {
    case CUEQ_F32: reinterpret_cast<float*>(p.out[which])[ch] = (float)v; break;
    case CUEQ_F64: reinterpret_cast<double*>(p.out[which])[ch] = (double)v; break;
    case CUEQ_BF16: reinterpret_cast<__nv_bfloat16*>(p.out[which])[ch] = __float2bfloat16_rn((float)v); break;
    default: reinterpret_cast<__half*>(p.out[which])[ch] = __float2half_rn((float)v); break;
  }
}

Kernel pick_kernel(int dtype, int mode, bool q8, bool mul_ir, bool backward) {
  switch (dtype) {
    case CUEQ_F32: return q8 ? pick_f32_codes(mode, mul_ir, backward) : pick_f32(mode, mul_ir, backward);
    case CUEQ_F64: return pick_f64(mode, mul_ir, backward);
    case CUEQ_BF16: return q8 ? pick_bf16_codes(mode, mul_ir, backward) : pick_bf16(mode, mul_ir, backward);
    default: return q8 ? pick_f16_codes(mode, mul_ir, backward) : pick_f16(mode, mul_ir, backward);
  }
}

int launch(const cueq_norm_args* a, bool backward, void* stream) {
  Params p;
  int grid = 0, smem = 0;
  if (!backward && a && a->stats) {                      // a backward pass is to come: it has to fit as well, and only long blocks do not
    if (int rc = check(a)) return rc;
    int longest = 0;
    for (int k = 0; k < a->num_blocks; ++k) { const int n = a->blocks[k].mul * a->blocks[k].dim; longest = n > longest ? n : longest; }
    if (longest > kSliceValues)
      if (int rc = fill(a, true, &p, &grid, &smem)) return rc;
  }
  if (int rc = fill(a, backward, &p, &grid, &smem)) return rc;
  const bool branch = a->mode & kBranch, norm = a->mode & kNorm;
  const int64_t width = p.dim_total, channels = p.channels;
  const bool q8 = a->codes != nullptr;
  auto operand = [&](const void* q, int64_t ld, int64_t w) { return q && (ld >= w || ld == 0 || a->rows <= 1); };
  if (branch && !a->scale) return cueq::fail("norm: null scale");
  if (norm && !a->weight) return cueq::fail("norm: null weight");
  if (gated(a) && !(backward && q8) && !operand(a->g, a->ldg, channels)) return cueq::fail("norm: gates are missing or their rows overlap");
  if (q8 && (a->ld_codes < code_layout(a, &p) || a->ld_codes % 16 || ((uintptr_t)a->codes & 15))) return cueq::fail("norm: rows of codes need %lld bytes, 16-byte aligned", (long long)code_layout(a, &p));
  if ((q8 || backward) && !a->stats) return cueq::fail("norm: null statistics");
  if ((uintptr_t)a->stats & 15) return cueq::fail("norm: statistics must be 16-byte aligned");
  if (!backward) {
    if (!operand(a->x, a->ldx, width) || (branch && !operand(a->y, a->ldy, width))) return cueq::fail("norm: an operand is missing or its rows overlap");
    if ((branch && !a->out) || (norm && !a->norm)) return cueq::fail("norm: null result");
  } else {
    if (!q8 && ((branch && !operand(a->y, a->ldy, width)) || (norm && !(again(a) ? operand(a->x, a->ldx, width) : operand(a->h, a->ldh, width))))) return cueq::fail("norm: a kept operand is missing or its rows overlap");
    if (norm ? !operand(a->gn, a->ldgn, width) : !operand(a->go, a->ldgo, width)) return cueq::fail("norm: a cotangent is missing or its rows overlap");
    if (a->mode == kBoth && a->go && !operand(a->go, a->ldgo, width)) return cueq::fail("norm: a cotangent's rows overlap");
    if ((branch && !a->dy) || (norm && !a->dx) || (gated(a) && !a->dg)) return cueq::fail("norm: null result");
    const int64_t need = 2 * (int64_t)grid * p.channels;
    if (a->parts_values < 0 && (a->dscale || a->dweight)) return cueq::fail("norm: the parameters' gradients need partial sums");
    if (a->rows && a->parts_values >= 0 && (!a->parts || a->parts_values < need)) return cueq::fail("norm: the parameters' gradients need room for %lld partial sums", (long long)need);
  }
  p.x = a->x; p.y = a->y; p.g = a->g; p.h = a->h; p.go = a->go; p.gn = a->gn;
  p.ldx = a->ldx; p.ldy = a->ldy; p.ldg = a->ldg; p.ldh = a->ldh; p.ldgo = a->ldgo; p.ldgn = a->ldgn;
  if (again(a)) { p.h = a->x; p.ldh = a->ldx; }
  p.s = a->scale; p.w = a->weight;
  p.out = a->out; p.norm = a->norm; p.dx = a->dx; p.dy = a->dy; p.dg = a->dg;
  p.codes = (signed char*)a->codes; p.ldc = a->ld_codes;
  p.stats = a->stats; p.parts = a->parts_values < 0 ? nullptr : a->parts;
  p.rows = a->rows; p.eps = a->eps; p.status = (int*)a->status;
  p.pdtype = a->param_dtype; p.mul_ir = a->mul_ir;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->rows) {
    const Kernel kernel = pick_kernel(a->dtype, a->mode, q8, a->mul_ir, backward);
    static cueq::PerDeviceFlag configured[4][3][2][2][2];
    cueq::PerDeviceFlag& flag = configured[a->dtype][a->mode - 1][q8][a->mul_ir != 0][backward];
    if (!flag.get()) {
      CUEQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerSm));
      flag.set();
    }
    kernel<<<grid, 32, smem, st>>>(p);
    CUEQ_CUDA_OK(cudaGetLastError());
  }
  if (!backward) return 0;
  SumParams s{a->parts, {branch ? a->dscale : nullptr, norm ? a->dweight : nullptr}, a->rows ? grid : 0, p.channels, a->param_dtype, p.status};
  if (!s.out[0] && !s.out[1]) return 0;
  const dim3 g((p.channels + kSumChannels - 1) / kSumChannels, 2), t(kSumChannels, kSumRows);
  if (a->dtype == CUEQ_F64) sum_kernel<double><<<g, t, 0, st>>>(s);
  else sum_kernel<float><<<g, t, 0, st>>>(s);
  CUEQ_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // namespace

extern "C" int64_t cueq_b200_norm_code_bytes(const cueq_norm_args* a) { return check(a) ? -1 : code_layout(a, nullptr); }
extern "C" int64_t cueq_b200_norm_stats(const cueq_norm_args* a) { return check(a) ? -1 : (int64_t)a->num_blocks * stats_per_item(a); }
extern "C" int64_t cueq_b200_norm_parts(const cueq_norm_args* a) {
  Params p;
  int grid, smem;
  return fill(a, true, &p, &grid, &smem) ? -1 : 2 * (int64_t)grid * p.channels;
}
extern "C" int cueq_b200_norm_forward(const cueq_norm_args* a, void* stream) { return launch(a, false, stream); }
extern "C" int cueq_b200_norm_backward(const cueq_norm_args* a, void* stream) { return launch(a, true, stream); }
