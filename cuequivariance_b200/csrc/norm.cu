// Host side of the norm kernels (norm_kernels.cuh): argument checks, the division of rows and irrep blocks among thread blocks,
// and the sum over thread blocks of the parameters' gradients.
#include <cstring>

#include "norm_kernels.cuh"

namespace {

using namespace cueq_norm;

constexpr int kSmemPerSm = 227 * 1024, kSms = 148;
constexpr int kStageBytes = 8192;        // rows are put together up to about this much per stage

int element_size(int dtype) { return dtype == CUEQ_F64 ? 8 : dtype == CUEQ_F32 ? 4 : 2; }
bool gated(const cueq_norm_args* a) { return a->gate != CUEQ_NORM_GATE_NONE && (a->mode & kBranch); }
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
    if (a->blocks[k].mul < 1 || a->blocks[k].dim < 1 || (int64_t)a->blocks[k].mul * a->blocks[k].dim > (1 << 24)) return cueq::fail("norm: bad irrep block %d", k);
  if (a->stats_stride && a->stats_stride != 8 && (a->stats_stride != 4 || (a->codes && a->mode == kBoth))) return cueq::fail("norm: bad stride of the statistics");
  if (!(a->eps > 0)) return cueq::fail("norm: eps must be positive");
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

// Divides the work.  A warp works alone on items of up to 256 values, two on up to 512, four on longer ones, but never more warps
// than there are groups of 32 channels.  Thread blocks are dealt to irrep blocks by their length; with few rows a stage holds
// fewer of them, so that they spread over the SMs.
int make_plan(const cueq_norm_args* a, bool backward, bool bulk, Params* p, int* grid, int* smem_bytes) {
  const bool q8 = a->codes != nullptr, gate = gated(a);
  const int size = element_size(a->dtype), msize = a->dtype == CUEQ_F64 ? 8 : 4, stat = stats_per_item(a) * msize;
  int64_t total_cost = 0;
  int smem = 0, dim_total = 0, channels = 0;
  for (int k = 0; k < a->num_blocks; ++k) {
    Blk& b = p->blk[k];
    b.mul = a->blocks[k].mul; b.dim = a->blocks[k].dim;
    b.off = dim_total; b.ch = channels;
    dim_total += b.mul * b.dim; channels += b.mul;
    const int n = b.mul * b.dim, groups = (b.mul + 31) / 32;
    b.wpi = n <= 256 || groups == 1 ? 1 : n <= 512 || groups == 2 ? 2 : 4;
    auto stage = [&](int rps) { return backward ? backward_stage(a->mode, q8, gate, size, b.mul, b.dim, rps, stat).total : forward_stage(a->mode, q8, gate, size, b.mul, b.dim, rps).total; };
    const int one = stage(1), ng = kWarps / b.wpi, head = head_bytes(msize, b.mul, backward, b.wpi);
    int rps = kStageBytes / one;
    rps = rps < ng ? ng : rps > 32 ? 32 : rps;
    while (rps > 1 && head + 2 * stage(rps) > kSmemPerSm / 4) --rps;
    b.rps = rps;
    const int need = head + (bulk ? 2 : 1) * stage(rps);
    smem = need > smem ? need : smem;
    total_cost += n + 96;
  }
  if (smem > kSmemPerSm) return -1;
  int occupancy = kSmemPerSm / (smem + 1024);
  occupancy = occupancy < 1 ? 1 : occupancy;
  const int most = msize == 8 ? 4 : 8;
  occupancy = occupancy > most ? most : occupancy;
  const int64_t ctas = (int64_t)kSms * occupancy;
  int at = 0;
  int64_t part = 0;
  for (int k = 0; k < a->num_blocks; ++k) {
    Blk& b = p->blk[k];
    int64_t share = ctas * (b.mul * b.dim + 96) / total_cost;
    share = share < 1 ? 1 : share;
    const int64_t spread = a->rows / share;
    if (b.rps > spread) b.rps = spread < 1 ? 1 : (int)spread;
    const int64_t units = (a->rows + b.rps - 1) / b.rps;
    b.ncta = (int)(share < units ? share : units);
    b.cta0 = at;
    at += b.ncta;
    b.part = part;
    part += (int64_t)b.ncta * b.mul;
  }
  p->nb = a->num_blocks; p->dim_total = dim_total; p->channels = channels;
  p->parts_len = part;
  *grid = at;
  *smem_bytes = smem;
  return 0;
}

bool aligned(const void* q, int64_t ld_bytes) { return !q || (((uintptr_t)q | (uintptr_t)ld_bytes) & 15) == 0; }

// Bulk copies want 16-byte boundaries and lengths.
bool bulk_ok(const cueq_norm_args* a) {
  const int size = element_size(a->dtype);
  int64_t dim = 0, channels = 0;
  for (int k = 0; k < a->num_blocks; ++k) {
    const int64_t n = (int64_t)a->blocks[k].mul * a->blocks[k].dim;
    if (n * size % 16 || (gated(a) && a->blocks[k].mul * size % 16)) return false;
    dim += n; channels += a->blocks[k].mul;
  }
  const void* operands[] = {a->x, a->y, a->g, a->h, a->go, a->gn};
  const int64_t lds[] = {a->ldx, a->ldy, a->ldg, a->ldh, a->ldgo, a->ldgn};
  for (int k = 0; k < 6; ++k) if (!aligned(operands[k], lds[k] * size)) return false;
  const void* rows[] = {a->out, a->norm, a->dx, a->dy};
  for (const void* q : rows) if (!aligned(q, dim * size)) return false;
  return aligned(a->dg, channels * size);
}

int fill(const cueq_norm_args* a, bool backward, Params* p, int* grid, int* smem) {
  std::memset(p, 0, sizeof(*p));
  if (int rc = check(a)) return rc;
  p->bulk = bulk_ok(a);
  int rc = make_plan(a, backward, p->bulk, p, grid, smem);
  if (rc && p->bulk) { p->bulk = 0; rc = make_plan(a, backward, false, p, grid, smem); }   // one stage at a time
  if (rc) return cueq::fail("norm: an irrep block does not fit into shared memory (%d bytes of %d)", *smem, kSmemPerSm);
  return 0;
}

// dscale, dweight: the thread blocks' sums of a channel, in order
struct SumParams {
  const void* parts;
  int64_t parts_len;
  void* out[2];
  int nb, channels, dtype;
  struct { int mul, ch, ncta; int64_t part; } blk[kMaxBlocks];
};
constexpr int kSumRows = 16;
template <class M>
__global__ void __launch_bounds__(32 * kSumRows) sum_kernel(const __grid_constant__ SumParams p) {
  __shared__ M partial[kSumRows][33];
  const int ch = blockIdx.x * 32 + threadIdx.x;
  const int which = blockIdx.y;
  M v = M(0);
  if (ch < p.channels && p.out[which]) {
    int k = 0;
    while (k + 1 < p.nb && ch >= p.blk[k + 1].ch) ++k;
    const M* src = reinterpret_cast<const M*>(p.parts) + which * p.parts_len + p.blk[k].part + (ch - p.blk[k].ch);
#pragma unroll 8
    for (int j = threadIdx.y; j < p.blk[k].ncta; j += kSumRows) v += src[(int64_t)j * p.blk[k].mul];
  }
  partial[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || ch >= p.channels || !p.out[which]) return;
  v = M(0);
#pragma unroll
  for (int j = 0; j < kSumRows; ++j) v += partial[j][threadIdx.x];
  switch (p.dtype) {
    case CUEQ_F32: reinterpret_cast<float*>(p.out[which])[ch] = (float)v; break;
    case CUEQ_F64: reinterpret_cast<double*>(p.out[which])[ch] = (double)v; break;
    case CUEQ_BF16: reinterpret_cast<__nv_bfloat16*>(p.out[which])[ch] = __float2bfloat16_rn((float)v); break;
    default: reinterpret_cast<__half*>(p.out[which])[ch] = __float2half_rn((float)v); break;
  }
}

Kernel pick_kernel(int dtype, int mode, bool q8, bool backward) {
  switch (dtype) {
    case CUEQ_F32: return pick_f32(mode, q8, backward);
    case CUEQ_F64: return pick_f64(mode, q8, backward);
    case CUEQ_BF16: return pick_bf16(mode, q8, backward);
    default: return pick_f16(mode, q8, backward);
  }
}

int launch(const cueq_norm_args* a, bool backward, void* stream) {
  Params p;
  int grid = 0, smem = 0;
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
    if (!q8 && ((branch && !operand(a->y, a->ldy, width)) || (norm && !operand(a->h, a->ldh, width)))) return cueq::fail("norm: a kept operand is missing or its rows overlap");
    if (norm ? !operand(a->gn, a->ldgn, width) : !operand(a->go, a->ldgo, width)) return cueq::fail("norm: a cotangent is missing or its rows overlap");
    if (a->mode == kBoth && a->go && !operand(a->go, a->ldgo, width)) return cueq::fail("norm: a cotangent's rows overlap");
    if ((branch && !a->dy) || (norm && !a->dx) || (gated(a) && !a->dg)) return cueq::fail("norm: null result");
    const int64_t need = 2 * p.parts_len;
    if (a->rows && (!a->parts || a->parts_values < need)) return cueq::fail("norm: the parameters' gradients need room for %lld partial sums", (long long)need);
  }
  p.x = a->x; p.y = a->y; p.g = a->g; p.h = a->h; p.go = a->go; p.gn = a->gn;
  p.ldx = a->ldx; p.ldy = a->ldy; p.ldg = a->ldg; p.ldh = a->ldh; p.ldgo = a->ldgo; p.ldgn = a->ldgn;
  p.s = a->scale; p.w = a->weight;
  p.out = a->out; p.norm = a->norm; p.dx = a->dx; p.dy = a->dy; p.dg = a->dg;
  p.codes = (signed char*)a->codes; p.ldc = a->ld_codes;
  p.stats = a->stats; p.parts = a->parts;
  p.rows = a->rows; p.eps = a->eps; p.status = (int*)a->status;
  p.ns = stats_per_item(a);
  p.pdtype = a->param_dtype; p.mul_ir = a->mul_ir;
  p.gate = branch ? a->gate : CUEQ_NORM_GATE_NONE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (a->rows) {
    const Kernel kernel = pick_kernel(a->dtype, a->mode, q8, backward);
    static cueq::PerDeviceFlag configured[4][3][2][2];
    cueq::PerDeviceFlag& flag = configured[a->dtype][a->mode - 1][q8][backward];
    if (!flag.get()) {
      CUEQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerSm));
      flag.set();
    }
    kernel<<<grid, kThreads, smem, st>>>(p);
    CUEQ_CUDA_OK(cudaGetLastError());
  }
  if (!backward) return 0;
  SumParams s;
  std::memset(&s, 0, sizeof(s));
  s.parts = a->parts; s.parts_len = p.parts_len;
  s.out[0] = branch ? a->dscale : nullptr;
  s.out[1] = norm ? a->dweight : nullptr;
  if (!s.out[0] && !s.out[1]) return 0;
  s.nb = p.nb; s.channels = p.channels; s.dtype = a->param_dtype;
  for (int k = 0; k < p.nb; ++k) { s.blk[k].mul = p.blk[k].mul; s.blk[k].ch = p.blk[k].ch; s.blk[k].ncta = a->rows ? p.blk[k].ncta : 0; s.blk[k].part = p.blk[k].part; }
  const dim3 g((p.channels + 31) / 32, 2), t(32, kSumRows);
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
  return fill(a, true, &p, &grid, &smem) ? -1 : 2 * p.parts_len;
}
extern "C" int cueq_b200_norm_forward(const cueq_norm_args* a, void* stream) { return launch(a, false, stream); }
extern "C" int cueq_b200_norm_backward(const cueq_norm_args* a, void* stream) { return launch(a, true, stream); }
