// Launchers of the Muon step (tmoe_muon.hpp).
#include <math.h>

#include <algorithm>
#include <vector>

#include "tmoe_muon.hpp"

namespace tmoe {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up(int64_t n, int64_t to) { return ceil_div(n, to) * to; }

struct Shape {
  int64_t batch, mp, np, chunks;
};
Shape shape_of(const tmoe_muon_tensor& t) {
  const int64_t lo = std::min(t.rows, t.cols), hi = std::max(t.rows, t.cols);
  return {t.batch, up(lo, 64), up(hi, 64), ceil_div(t.rows * t.cols, dev::kMuonChunk)};
}
bool empty(const tmoe_muon_tensor& t) { return t.batch == 0 || t.rows == 0 || t.cols == 0; }

// The workspace: the table, the chunks' sums, then for each tensor X and X^T twice, A and B
struct Layout {
  int64_t count = 0, chunks = 0, sums, planes, total;
};
Layout layout_of(const tmoe_muon_tensor* t, int64_t count) {
  Layout l;
  int64_t halves = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (empty(t[i])) continue;
    const Shape s = shape_of(t[i]);
    ++l.count;
    l.chunks += s.batch * s.chunks;
    halves += s.batch * (8 * s.mp * s.np + 4 * s.mp * s.mp);
  }
  l.sums = up(l.count * (int64_t)sizeof(MuonDesc), 256);
  l.planes = up(l.sums + l.chunks * 4, 256);
  l.total = l.planes + 2 * halves;
  return l;
}

template <int BT, class T>
void gemm(int phase, const MuonArgs& a, unsigned groups, hipStream_t st) {
  const dim3 grid(groups), block(dev::kMuonThreads);
  switch (phase) {
    case dev::kMuonGram: hipLaunchKernelGGL((dev::k_muon_gemm<BT, dev::kMuonGram, uint16_t>), grid, block, 0, st, a); break;
    case dev::kMuonPoly: hipLaunchKernelGGL((dev::k_muon_gemm<BT, dev::kMuonPoly, uint16_t>), grid, block, 0, st, a); break;
    case dev::kMuonApply: hipLaunchKernelGGL((dev::k_muon_gemm<BT, dev::kMuonApply, uint16_t>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((dev::k_muon_gemm<BT, dev::kMuonLast, T>), grid, block, 0, st, a); break;
  }
}

}  // namespace

size_t muon_workspace_bytes(const tmoe_muon_tensor* t, int64_t count) {
  const Layout l = layout_of(t, count);
  return l.count ? (size_t)l.total : 0;
}

hipError_t muon(const tmoe_muon_tensor* t, int64_t count, const tmoe_muon_step_args& s, void* ws, hipStream_t st) {
  const Layout l = layout_of(t, count);
  if (!l.count) return hipSuccess;
  const bool bf16 = s.dtype == TMOE_BF16;
  // tiles of 128 where they fill the chip
  int64_t wide = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (empty(t[i])) continue;
    const Shape q = shape_of(t[i]);
    wide += q.batch * ceil_div(q.mp, 128) * ceil_div(q.np, 128);
  }
  const int64_t bt = wide >= 512 ? 128 : 64;
  char* base = static_cast<char*>(ws);
  MuonChunkArgs c{};
  c.table = reinterpret_cast<MuonDesc*>(base);
  c.sums = reinterpret_cast<float*>(base + l.sums);
  c.mu = (float)s.momentum;
  c.nesterov = s.nesterov;
  uint16_t* plane = reinterpret_cast<uint16_t*>(base + l.planes);
  uint32_t chunk0 = 0, tile0 = 0, sym0 = 0, app0 = 0, done = 0;
  auto flush = [&]() {
    if (!c.count) return hipSuccess;
    c.first = (int)done;
    const dim3 grid(chunk0 - c.t[0].chunk0), block(dev::kMuonThreads);
    if (bf16) hipLaunchKernelGGL(dev::k_muon_momentum<uint16_t>, grid, block, 0, st, c);
    else hipLaunchKernelGGL(dev::k_muon_momentum<float>, grid, block, 0, st, c);
    done += c.count;
    c.count = 0;
    return hipGetLastError();
  };
  static_assert(sizeof(MuonChunkArgs) <= 4096, "a launch's arguments");
  for (int64_t i = 0; i < count; ++i) {
    if (empty(t[i])) continue;
    const Shape q = shape_of(t[i]);
    MuonDesc& d = c.t[c.count++];
    d.p = t[i].p; d.g = t[i].g; d.m = t[i].m;
    const int64_t xs = 2 * q.batch * q.mp * q.np, as = 2 * q.batch * q.mp * q.mp;
    for (int k = 0; k < 2; ++k) {
      d.x[k] = plane; plane += xs;
      d.xt[k] = plane; plane += xs;
    }
    d.a = plane; plane += as;
    d.b = plane; plane += as;
    d.rows = (int)t[i].rows; d.cols = (int)t[i].cols; d.mp = (int)q.mp; d.np = (int)q.np;
    d.chunk0 = chunk0; d.chunks = (uint32_t)q.chunks;
    d.tile0 = tile0; d.sym0 = sym0; d.app0 = app0;
    d.rate = s.write_only ? -1.f
                          : (float)(s.lr * s.update_rms * sqrt((double)std::max(t[i].rows, t[i].cols)));
    chunk0 += (uint32_t)(q.batch * q.chunks);
    tile0 += (uint32_t)(q.batch * (q.mp / 64) * (q.np / 64));
    const int64_t tm = ceil_div(q.mp, bt), tn = ceil_div(q.np, bt);
    sym0 += (uint32_t)(q.batch * tm * (tm + 1) / 2);
    app0 += (uint32_t)(q.batch * tm * tn);
    if (c.count == kMuonTensors)
      if (hipError_t e = flush(); e != hipSuccess) return e;
  }
  if (hipError_t e = flush(); e != hipSuccess) return e;
  MuonArgs a{};
  a.table = c.table; a.sums = c.sums; a.count = (int)l.count; a.nesterov = s.nesterov;
  a.mu = c.mu; a.eps = (float)s.eps;
  a.a = (float)s.coefficients[0]; a.b = (float)s.coefficients[1]; a.c = (float)s.coefficients[2];
  a.keep = s.write_only ? 0.f : (float)(1.0 - s.lr * s.weight_decay);
  if (bf16) hipLaunchKernelGGL(dev::k_muon_start<uint16_t>, dim3(tile0), dim3(dev::kMuonThreads), 0, st, a);
  else hipLaunchKernelGGL(dev::k_muon_start<float>, dim3(tile0), dim3(dev::kMuonThreads), 0, st, a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  for (int i = 0; i < s.steps; ++i) {
    for (int phase = 0; phase < 3; ++phase) {
      const int k = phase == dev::kMuonApply && i + 1 == s.steps ? dev::kMuonLast : phase;
      const unsigned groups = phase < dev::kMuonApply ? sym0 : app0;
      if (bt == 128) bf16 ? gemm<128, uint16_t>(k, a, groups, st) : gemm<128, float>(k, a, groups, st);
      else bf16 ? gemm<64, uint16_t>(k, a, groups, st) : gemm<64, float>(k, a, groups, st);
      if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    a.cur ^= 1;
  }
  return hipSuccess;
}

}  // namespace tmoe
