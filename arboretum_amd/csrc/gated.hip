// The gated layer and its gradient: checks of arguments, and how the products are cut up (the kernels: gated_kernels.h).
#include <algorithm>

#include "gated_launch.h"
#include "operators_device.h"

namespace arb {
namespace {

constexpr int kPlaces = 256 * SmallTile::kEach;

// A product of `rows` x `columns` (`batch` of them) over `blocks` blocks of k's; half: a tile has half as many columns.  Large tiles, which read the LDS less for
// each product, where they fill the chip, are not mostly beyond its columns, and have k's enough that their results are not most of the work (the layer
// itself, small and large: 50000 x 100 x 300 27.9 and 31.4 us, 100000 x 256 x 512 77.5 and 78.1, 20000 x 1024 x 2048 173 and 151).  Else small ones, and few of them share out
// their k's until `places` have one (of kPlaces, the halves of the CUs): at least `least` blocks to a share, and 24 where there are more than 64 shares, whose sums are written and read
// again (200000 x 16 x 64, the gradient's last product in 64 and 128 shares: 114 and 105 us in all, float32 375 and 279; 100003 x 64 x 256 150 and 154).
ProductCut CutOf(long long rows, long long columns, int half, long long batch, long long blocks, long long least, int places) {
  const auto tiles = [&](long long i, long long j) { return Pieces(rows, i) * Pieces(columns, j / half) * batch; };
  const long long large = tiles(LargeTile::kI, LargeTile::kJ), small = tiles(SmallTile::kI, SmallTile::kJ);
  ProductCut c;
  c.large = large >= 200 && columns > SmallTile::kJ / half && blocks > 2;
  const long long free = c.large ? 256 / large : places / std::max<long long>(small, 1);
  const long long most = std::max<long long>(1, std::min(free, std::max(std::min(blocks / least, 64ll), std::min(blocks / 24, 128ll))));
  c.split_blocks = std::max<long long>(1, Pieces(blocks, most));
  c.splits = std::max<long long>(1, Pieces(blocks, c.split_blocks));
  c.tiles = (c.large ? large : small) * c.splits;
  return c;
}

// Bytes taken one after the other, each piece on 256.
struct Room {
  size_t bytes = 0;
  size_t Take(size_t more) {
    const size_t at = bytes;
    bytes += (more + 255) / 256 * 256;
    return at;
  }
};

// Rows whose chunks are not aligned come through registers into small tiles, a block at a time; copies of x and both weights are read and written once.  For the
// gradient (300 x 4094 x 4098 with the layer itself: 251 us without, 186 with copies; 100 x 1002 x 1004 68 and 44) the copies are always less.
// There is room for them by the width alone, since whoever asks for the bytes says no more: rows of whole chunks that lie between the places of such go through registers
// whatever their number (8192 x 4096 x 16384 bf16, one element between rows and none: layer 3576 and 1883 us, gradient 5657 and 3686; 1000 x 768 x 2048 35 and 34, 63 and 40).
LayerPad PadOf(long long rows, int dim, int hidden, size_t item, Room *room) {
  LayerPad p{0, 0, 0, 0};
  if (dim * item % 16 == 0 || rows == 0) return p;
  p.stride = Pieces(dim, 64) * 64;
  p.x = room->Take((size_t)rows * p.stride * item);
  p.w_gate = room->Take((size_t)hidden * p.stride * item);
  p.w_up = room->Take((size_t)hidden * p.stride * item);
  return p;
}

// Whether the layer itself, which reads its weights along k, copies too, by a line through the times that follow: a block through registers takes 1.3 us more, the last one of a row three times that, copies a launch of
// 5 us and their bytes at 5 TB/s (us without and with: 40 x 4095 x 16383 92 and 175, 300 x 4095 x 4097 66 and 69, 500 x 1001 x 1003 20 and 18, 8191 x 1001 x 1003
// 57 and 42, 100,003 x 63 x 255 70 and 49, 280 x 7353 x 11442 380 and 297).
bool CopiesForward(const ProductCut &c, long long rows, int dim, int hidden, size_t item) {
  const long long turns = Pieces(Pieces(rows, SmallTile::kI) * Pieces(hidden, SmallTile::kJ / 2) * c.splits, kPlaces);
  return 1.3 * turns * (c.split_blocks + 2) > 5.0 + 2.0 * (rows + 2.0 * hidden) * dim * item / 5.0e6;
}

void CheckLayerSizes(long long rows, int dim, int hidden, int type) {
  CheckType(type);
  if (rows < 0 || rows >= (1ll << 31)) throw std::runtime_error("bad number of rows");
  if (dim < 1 || dim > (1 << 24)) throw std::runtime_error("bad dimension");
  if (hidden < 1 || hidden > (1 << 24)) throw std::runtime_error("bad hidden dimension");
}

GatedPlan PlanOf(long long rows, int dim, int hidden, int type) {
  const size_t item = ElementBytes(type);
  GatedPlan p;
  Room room;
  p.few = rows <= kFewRows;
  p.out = CutOf(rows, hidden, 2, 1, Pieces(dim * item, kLineBytes), 4, kPlaces);
  p.pad = CopiesForward(p.out, rows, dim, hidden, item) ? PadOf(rows, dim, hidden, item, &room) : LayerPad{0, 0, 0, 0};
  p.partial = room.Take(p.out.splits > 1 ? (size_t)p.out.splits * rows * Pieces(hidden, kScaleGroup) * kWaveJ * sizeof(float) : 0);
  p.bytes = room.bytes;
  return p;
}

GatedGradPlan GradPlanOf(long long rows, int dim, int hidden, int type) {
  const size_t item = ElementBytes(type);
  GatedGradPlan p;
  Room room;
  p.d_stride = Pieces(hidden, 64) * 64;
  // Both products at once where a half of the places is enough for each, one after the other elsewhere.
  for (const int places : {kPlaces / 2, kPlaces}) {
    p.x = CutOf(rows, dim, 1, 1, 2 * Pieces(hidden * item, kLineBytes), 8, places);
    p.w = CutOf(hidden, dim, 1, 2, Pieces(rows * item, kLineBytes), 4, places);
    p.together = !p.x.large && !p.w.large && p.x.tiles + p.w.tiles <= kPlaces;
    if (p.together) break;
  }
  p.d_gate = room.Take((size_t)rows * p.d_stride * item);
  p.d_up = room.Take((size_t)rows * p.d_stride * item);
  p.range = room.Take(type == kFloat16 && rows > 0 ? (1 + kRangeGroups) * sizeof(float) : 0);
  p.pad = PadOf(rows, dim, hidden, item, &room);
  p.x_partial = room.Take(p.x.splits > 1 ? (size_t)p.x.splits * rows * dim * sizeof(float) : 0);
  p.w_partial = room.Take(p.w.splits > 1 ? (size_t)p.w.splits * 2 * hidden * dim * sizeof(float) : 0);
  p.bytes = room.bytes;
  return p;
}

void CheckStride(long long stride, long long width, long long rows, const char *what) {
  if (stride < 0 || stride >= (1ll << 31) || (rows > 1 && stride < width)) throw std::runtime_error(std::string("bad stride of ") + what);
}

// (checks what both directions take; kept: whether gate and up must be there)
void CheckLayer(const GatedLayer &l, bool kept, size_t need) {
  CheckLayerSizes(l.rows, l.dim, l.hidden, l.type);
  if (l.activation != kSilu && l.activation != kGelu) throw std::runtime_error("unknown activation");
  CheckStride(l.x_stride, 0, l.rows, "x");
  CheckStride(l.w_stride, 0, l.hidden, "the weights");
  if (!l.w_gate || !l.w_up || (l.rows > 0 && !l.x)) throw std::runtime_error("null pointer argument");
  if ((l.gate == nullptr) != (l.up == nullptr) || (l.gate_scales == nullptr) != (l.up_scales == nullptr)) throw std::runtime_error("gate and up go together");
  if (l.gate_scales && !l.gate) throw std::runtime_error("scales without gate and up");
  if (kept && l.rows > 0 && !l.gate) throw std::runtime_error("null pointer argument");
  if (l.gate) CheckStride(l.kept_stride, l.hidden, l.rows, "gate and up");
  const size_t item = ElementBytes(l.type);
  CheckAligned(l.x, item, "x");
  CheckAligned(l.w_gate, item, "w_gate");
  CheckAligned(l.w_up, item, "w_up");
  if (!l.gate_scales) CheckAligned(l.gate, item, "gate"), CheckAligned(l.up, item, "up");
  CheckAligned(l.gate_scales, 4, "gate_scales");
  CheckAligned(l.up_scales, 4, "up_scales");
  if (need > 0) {
    if (!l.work) throw std::runtime_error("null pointer argument");
    CheckAligned(l.work, 16, "work");
    if (l.work_bytes < need) throw std::runtime_error("work memory is too small: " + std::to_string(need) + " bytes are needed");
  }
}

}  // namespace

size_t GatedBytes(long long rows, int dim, int hidden, int type) {
  CheckLayerSizes(rows, dim, hidden, type);
  return PlanOf(rows, dim, hidden, type).bytes;
}

void Gated(const GatedArgs &a) {
  const GatedLayer &l = a.layer;
  const GatedPlan plan = (CheckLayerSizes(l.rows, l.dim, l.hidden, l.type), PlanOf(l.rows, l.dim, l.hidden, l.type));
  const size_t need = plan.few && !l.gate_scales ? 0 : plan.bytes;  // (few rows go without, but for codes, whose scales stand for 64 columns)
  CheckLayer(l, false, need);
  CheckStride(a.out_stride, l.hidden, l.rows, "out");
  CheckAligned(a.out, ElementBytes(l.type), "out");
  if (l.rows == 0) return;
  if (!a.out) throw std::runtime_error("null pointer argument");
  const size_t item = ElementBytes(l.type), kept = l.gate_scales ? 1 : item;
  const long long scales = l.rows * Pieces(l.hidden, kScaleGroup) * 4;
  CheckApart({{a.out, l.rows, a.out_stride, l.hidden, item}, {l.gate, l.rows, l.kept_stride, l.hidden, kept}, {l.up, l.rows, l.kept_stride, l.hidden, kept},
              {l.gate_scales, scales}, {l.up_scales, scales}, {l.work, (long long)need}},
             {{l.x, l.rows, l.x_stride, l.dim, item}, {l.w_gate, l.hidden, l.w_stride, l.dim, item}, {l.w_up, l.hidden, l.w_stride, l.dim, item}});
  OnDeviceOf device(a.out);
  WithType(l.type, [&](auto type) { RunGated<decltype(type)>(a, plan); });
}

size_t GatedGradBytes(long long rows, int dim, int hidden, int type) {
  CheckLayerSizes(rows, dim, hidden, type);
  return GradPlanOf(rows, dim, hidden, type).bytes;
}

void GatedGrad(const GatedGradArgs &a) {
  const GatedLayer &l = a.layer;
  const GatedGradPlan plan = (CheckLayerSizes(l.rows, l.dim, l.hidden, l.type), GradPlanOf(l.rows, l.dim, l.hidden, l.type));
  CheckLayer(l, true, plan.bytes);
  if ((a.grad_w_gate == nullptr) != (a.grad_w_up == nullptr)) throw std::runtime_error("the gradients of both weights go together");
  const size_t item = ElementBytes(l.type);
  CheckAligned(a.grad_out, item, "grad_out");
  CheckAligned(a.grad_x, item, "grad_x");
  CheckAligned(a.grad_w_gate, item, "grad_w_gate");
  CheckAligned(a.grad_w_up, item, "grad_w_up");
  CheckStride(a.grad_out_stride, 0, l.rows, "grad_out");
  if (a.grad_x) CheckStride(a.grad_x_stride, l.dim, l.rows, "grad_x");
  if (a.grad_w_gate) CheckStride(a.grad_w_stride, l.dim, l.hidden, "the weights' gradients");
  if (l.rows > 0 && !a.grad_out) throw std::runtime_error("null pointer argument");
  if (!a.grad_w_gate && (!a.grad_x || l.rows == 0)) return;
  const size_t kept = l.gate_scales ? 1 : item;
  const long long scales = l.rows * Pieces(l.hidden, kScaleGroup) * 4;
  CheckApart({{a.grad_x, l.rows, a.grad_x_stride, l.dim, item}, {a.grad_w_gate, l.hidden, a.grad_w_stride, l.dim, item},
              {a.grad_w_up, l.hidden, a.grad_w_stride, l.dim, item}, {l.work, (long long)plan.bytes}},
             {{a.grad_out, l.rows, a.grad_out_stride, l.hidden, item}, {l.x, l.rows, l.x_stride, l.dim, item}, {l.w_gate, l.hidden, l.w_stride, l.dim, item},
              {l.w_up, l.hidden, l.w_stride, l.dim, item}, {l.gate, l.rows, l.kept_stride, l.hidden, kept}, {l.up, l.rows, l.kept_stride, l.hidden, kept},
              {l.gate_scales, scales}, {l.up_scales, scales}});
  OnDeviceOf device(a.grad_w_gate ? a.grad_w_gate : a.grad_x);
  WithType(l.type, [&](auto type) { RunGatedGrad<decltype(type)>(a, plan); });
}

}  // namespace arb
