// Launchers of the Muon step (tmoe_muon.hpp).
#include <math.h>

#include <algorithm>

#include "tmoe_muon.hpp"

namespace tmoe {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up(int64_t n, int64_t to) { return ceil_div(n, to) * to; }

bool empty(const tmoe_muon_tensor& t) { return t.batch == 0 || t.rows == 0 || t.cols == 0; }

struct Shape {
  int64_t rp, cp, m, chunks, halves;   // of a matrix
};
Shape shape_of(const tmoe_muon_tensor& t) {
  Shape s;
  s.rp = up(t.rows, 64);
  s.cp = up(t.cols, 64);
  s.m = t.rows > t.cols ? s.cp : s.rp;
  s.chunks = ceil_div(t.rows * t.cols, dev::kMuonChunk);
  s.halves = 4 * s.rp * s.cp + 4 * s.m * s.m;
  return s;
}

// Tensors are stepped in groups, one after another in one workspace; a tensor that is larger is a
// group of its own. Planes that the memory-side cache holds (256 MB) gain nothing: the 66 layers of
// the reference model took 22.1 ms in groups of 160 MB, 18.6 of 320, 17.0 of 640, 15.8 of 1280 and
// without a limit (48 tensors each), since each launch has a start and an end.
constexpr int64_t kGroupBytes = (int64_t)1280 << 20;
constexpr int64_t kTableBytes = (kMuonTensors * (int64_t)sizeof(MuonDesc) + 255) / 256 * 256;
// the tensors from i on that are a group: their end, and what they need
struct Group {
  int64_t end, chunks, halves;
  int64_t planes_at() const { return up(kTableBytes + chunks * 8, 256); }
  int64_t bytes() const { return planes_at() + 2 * halves; }
};
Group group_from(const tmoe_muon_tensor* t, int64_t i, int64_t count) {
  Group g{i, 0, 0};
  for (int n = 0; g.end < count && n < kMuonTensors; ++g.end) {
    if (empty(t[g.end])) continue;
    const Shape s = shape_of(t[g.end]);
    const int64_t halves = t[g.end].batch * s.halves;
    if (n && 2 * (g.halves + halves) > kGroupBytes) break;
    g.halves += halves;
    g.chunks += t[g.end].batch * s.chunks;
    ++n;
  }
  return g;
}

// 64 x 64: 16 KB stages, two work-groups of four waves to a compute unit. Three stages, and three
// work-groups, took 129 us a step against 124 (six small matrices) and 406 against 389 (up to 1024 x 2304).
using Small = dev::MuonTile<64, 64, 2, 2, 4>;
// 128 x 128, for the symmetric products eight waves in two groups, for the third product two
// work-groups of four waves, one of which has its products while the other starts or stores: of 96 of
// 256 x 512 beside six wide ones 745 us a step against 782 with 256 x 128 of eight waves (4.63 ms against
// 4.48 for one of 4096 x 4096), and 762 with such work-groups for all three.
using Square = dev::MuonTile<128, 128, 4, 2, 4>;      // 32 KB stages
using Pair = dev::MuonTile<128, 128, 2, 2, 2>;        // 32 KB stages

template <class TL, int PHASE, class T = uint16_t>
void launch(const MuonArgs& a, unsigned groups, hipStream_t st) {
  hipLaunchKernelGGL((dev::k_muon_gemm<TL, PHASE, T>), dim3(groups), dim3(TL::kThreads), 0, st, a);
}
template <class TL>
void launch_symmetric(int phase, const MuonArgs& a, unsigned groups, unsigned sums, hipStream_t st) {
  if (phase == dev::kMuonPoly) return launch<TL, dev::kMuonPoly>(a, groups, st);
  launch<TL, dev::kMuonGram>(a, groups, st);
  if (sums) hipLaunchKernelGGL((dev::k_muon_sum<TL>), dim3(sums), dim3(64), 0, st, a);
}
template <class TL>
void launch_apply(bool last, bool bf16, const MuonArgs& a, unsigned groups, hipStream_t st) {
  if (!last) launch<TL, dev::kMuonApply>(a, groups, st);
  else if (bf16) launch<TL, dev::kMuonLast, uint16_t>(a, groups, st);
  else launch<TL, dev::kMuonLast, float>(a, groups, st);
}

}  // namespace

size_t muon_workspace_bytes(const tmoe_muon_tensor* t, int64_t count) {
  int64_t most = 0;
  for (int64_t i = 0; i < count;) {
    const Group g = group_from(t, i, count);
    if (g.halves) most = std::max(most, g.bytes());
    i = g.end;
  }
  return (size_t)most;
}

hipError_t muon(const tmoe_muon_tensor* t, int64_t count, const tmoe_muon_step_args& s, void* ws, hipStream_t st) {
  static_assert(sizeof(MuonFirstArgs) <= 4096, "a launch's arguments");
  const bool bf16 = s.dtype == TMOE_BF16;
  const dim3 block(dev::kMuonThreads);
  MuonFirstArgs first{};
  MuonArgs& a = first.a;
  a.t = static_cast<MuonDesc*>(ws);
  a.sums = reinterpret_cast<double*>(static_cast<char*>(ws) + kTableBytes);
  a.mu = (float)s.momentum; a.eps = (float)s.eps; a.nesterov = s.nesterov; a.write_only = s.write_only;
  a.a = (float)s.coefficients[0]; a.b = (float)s.coefficients[1]; a.c = (float)s.coefficients[2];
  a.keep = (float)(1.0 - s.lr * s.weight_decay);
  for (int64_t i = 0; i < count;) {
    const Group g = group_from(t, i, count);
    uint16_t* plane = reinterpret_cast<uint16_t*>(static_cast<char*>(ws) + g.planes_at());
    // Tiles of 128 x 128 where X has one for each compute unit and half of A some for every fourth. us a
    // step, 128 against 64: 2048 x 2048 (136 of A, 256 of X) 762 and 987, 6144 x 1536 (78, 576) 1151 and 1333, 32
    // of 256 x 512 (96, 256) 208 and 218; 1536 x 1536 (78, 144) 590 and 499, 1024 x 4096 (36, 256) 450 and
    // 434, 16 of 256 x 512 (48, 128) 181 and 152. Between 36 and 78 of A, and 144 and 256 of X, nothing was.
    int64_t pairs128 = 0, square = 0;
    for (int64_t k = i; k < g.end; ++k) {
      const Shape q = shape_of(t[k]);
      if (empty(t[k])) continue;
      const int64_t side = ceil_div(q.m, 128);
      pairs128 += t[k].batch * side * (side + 1) / 2;
      square += t[k].batch * ceil_div(q.rp, 128) * ceil_div(q.cp, 128);
    }
    const int64_t bt = pairs128 >= 72 && square >= 256 ? 128 : 64;
    // The Gram products' summed axes are cut into slices of about what each work-group that the
    // chip holds has to do in the mean: a long one alone would keep the rest waiting. For what the sum
    // costs that mean is taken as 14 K tiles at least (16 of 128 x 128), and an axis cut evenly into the
    // fewest slices of no more: 16 K tiles are two of 8, 32 three of 11, 11 and 10. A step of nine small
    // matrices takes 135 us so and 140 with 8 or with 16 as the least; between those only 14 was measured.
    int64_t work = 0;
    for (int64_t k = i; k < g.end; ++k) {
      if (empty(t[k])) continue;
      const Shape q = shape_of(t[k]);
      const int64_t side = ceil_div(q.m, bt);
      work += t[k].batch * side * (side + 1) / 2 * (std::max(q.rp, q.cp) / dev::kMuonK);
    }
    const int64_t mean = std::max(ceil_div(work, bt == 128 ? 256 : 512), bt == 128 ? (int64_t)16 : (int64_t)14);
    uint32_t chunk0 = 0, tile0 = 0, gram0 = 0, sum0 = 0, sym0 = 0, app0 = 0;
    a.count = a.cur = 0;
    for (; i < g.end; ++i) {
      if (empty(t[i])) continue;
      const Shape q = shape_of(t[i]);
      MuonDesc& d = first.t[a.count++];
      d.p = t[i].p; d.g = t[i].g; d.m = t[i].m;
      d.planes = plane;
      plane += t[i].batch * q.halves;
      d.rows = (int)t[i].rows; d.cols = (int)t[i].cols;
      d.chunk0 = chunk0; d.chunks = (uint32_t)q.chunks;
      d.tile0 = tile0; d.gram0 = gram0; d.sum0 = sum0; d.sym0 = sym0; d.app0 = app0;
      d.rate = s.write_only ? -1.f
                            : (float)(s.lr * s.update_rms * sqrt((double)std::max(t[i].rows, t[i].cols)));
      const int64_t side = ceil_div(q.m, bt), pairs = side * (side + 1) / 2;
      const int64_t all = std::max(q.rp, q.cp) / dev::kMuonK;
      // (the slices' sums have to find room in X')
      const int64_t n = std::max(std::min(ceil_div(all, mean), q.rp * q.cp / (pairs * bt * bt)), (int64_t)1);
      d.slice_tiles = (int)ceil_div(all, n);
      d.slices = (int)ceil_div(all, d.slice_tiles);
      gram0 += (uint32_t)(t[i].batch * pairs * d.slices);
      if (d.slices > 1) sum0 += (uint32_t)(t[i].batch * pairs * (bt / 32) * (bt / 32));
      chunk0 += (uint32_t)(t[i].batch * q.chunks);
      tile0 += (uint32_t)(t[i].batch * ceil_div(q.rp * q.cp, dev::kMuonChunk));
      sym0 += (uint32_t)(t[i].batch * pairs);
      app0 += (uint32_t)(t[i].batch * ceil_div(q.rp, bt) * ceil_div(q.cp, bt));
    }
    if (!a.count) continue;
    if (bf16) {
      hipLaunchKernelGGL(dev::k_muon_momentum<uint16_t>, dim3(chunk0), block, 0, st, first);
      hipLaunchKernelGGL(dev::k_muon_start<uint16_t>, dim3(tile0), block, 0, st, a);
    } else {
      hipLaunchKernelGGL(dev::k_muon_momentum<float>, dim3(chunk0), block, 0, st, first);
      hipLaunchKernelGGL(dev::k_muon_start<float>, dim3(tile0), block, 0, st, a);
    }
    for (int k = 0; k < s.steps; ++k) {
      for (int phase : {dev::kMuonGram, dev::kMuonPoly}) {
        const unsigned groups = phase == dev::kMuonGram ? gram0 : sym0;
        if (bt == 128) launch_symmetric<Square>(phase, a, groups, sum0, st);
        else launch_symmetric<Small>(phase, a, groups, sum0, st);
      }
      const bool last = k + 1 == s.steps;
      if (bt == 128) launch_apply<Pair>(last, bf16, a, app0, st);
      else launch_apply<Small>(last, bf16, a, app0, st);
      a.cur ^= 1;
    }
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tmoe
