// C entries of linear maps and feed-forward parts: checks, workspaces, and which kernels run (nd_linear.hpp).
#include "../../include/nextdoor_amd.h"

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "nd_errors.hpp"
#include "nd_linear.hpp"

namespace nd {

namespace {

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// ---- which tiles, and how many shares of a sum -------------------------------------------------------------------

// An estimate of a product's time in us, from what its workgroups take for a round of 64 places where a compute unit here and there
// has one, where each has one, and where each has as many as it holds; and beside the rounds.  (60 products of 1021 to 20483 rows, each
// timed with every shape: what the estimate takes is the fastest or 2 % off, where sums are not cut.)
struct ShapeCost {
  int m, n, at_once;  // rows of C, columns of C, workgroups that the GPU holds at a time
  double lone, one, full, once;
};
constexpr ShapeCost kShapes[4] = {{256, 256, 256, 1.05, 1.5, 1.5, 10.0},
                                  {128, 128, 512, 0.56, 0.6, 0.87, 4.0},
                                  {64, 64, 768, 0.32, 0.4, 0.5, 3.0},
                                  {256, 192, 256, 0.9, 1.2, 1.2, 9.0}};
constexpr int kMostShares = 128;
constexpr int64_t kRowsAlone = 256;     // whose sums one workgroup makes: less than another launch, which adds up shares, costs
constexpr int64_t kCaches = 32 << 20;  // bytes of the L2 caches of all dies
// us of adding sums: a launch in a forward pass, a part of one in a backward pass; bytes a us of them, written and read again; us of a launch
constexpr double kJoin = 4.0, kJoinPart = 2.0, kJoinRate = 8e6, kLaunch = 3.0;

double time_of(const ShapeCost& c, int64_t groups, int64_t rounds) {
  const int64_t full = groups / c.at_once, rest = groups % c.at_once;
  const double last = rest <= 256 ? c.lone + (c.one - c.lone) * rest / 256 : c.one + (c.full - c.one) * (rest - 256) / (c.at_once - 256);
  return full * (rounds * c.full + c.once) + (rest ? rounds * last + c.once : 0);
}

// A product C [m][n], sums over k.
struct Task {
  int64_t m, n, k;
  After after;
};
// Into how many shares its sums may be cut with tiles of one shape.
struct Shares {
  static constexpr int kMost = 12;
  int n = 0;
  int shares[kMost];
  int64_t groups[kMost], rounds[kMost];  // workgroups; rounds of each
  double joined[kMost];                  // us of adding the shares
};
void shares_of(const Task& t, const ShapeCost& c, Shares& s) {
  const int64_t rounds = std::max<int64_t>(1, (t.k + 63) / 64), columns = t.after == After::kGated ? 2 * t.n : t.n;
  const int64_t tiles = ((t.m + c.m - 1) / c.m) * ((columns + c.n - 1) / c.n);
  const int most = t.after == After::kSlope ? 1 : kMostShares;
  for (int want = 1; want <= most && s.n < Shares::kMost; want = want < 4 ? want + 1 : want * 3 / 2) {
    if (want > 1 && tiles * want > 4 * c.at_once) break;
    const int64_t each = (rounds + want - 1) / want;
    if ((rounds + each - 1) / each != want) continue;
    s.shares[s.n] = want;
    s.groups[s.n] = tiles * want;
    s.rounds[s.n] = each;
    s.joined[s.n++] = want > 1 ? (t.after == After::kPlain ? kJoinPart : kJoin) + (double)want * t.m * columns * 8 / kJoinRate : 0;
  }
}
struct Estimate {
  LinearPlan plan;
  double time;
};
// Columns of a pair's two halves alternate by 32, and a slope is read for 64 at a time: neither divides a wave's part of a narrow tile.
bool makes(int shape, After after) { return shape != 3 || (after != After::kGated && after != After::kSlope); }
Estimate estimate(const Task& t) {
  Estimate best = {{}, INFINITY};
  for (int shape = 0; shape < 4; ++shape) {
    Shares s;
    shares_of(t, kShapes[shape], s);
    for (int i = 0; i < s.n; ++i) {
      if (s.shares[i] == 1 && !makes(shape, t.after)) continue;
      const double time = time_of(kShapes[shape], s.groups[i], s.rounds[i]) + s.joined[i];
      if (time < best.time) best = {{shape, s.shares[i], (int)s.rounds[i] * 64}, time};
    }
  }
  // Large tiles for as many rows as they fill whole turns of the compute units with, another shape for the rows behind those, where
  // that is estimated to take a sixteenth less (what the estimate is off by; 9000 x 2000 -> 2048: 91 us for 112, its gradient of x 77 for
  // 89; 20000 x 4096 -> 1024: 148 for 155; 8192 x 2048 x 11264 by columns, estimated at 303 for 321: no difference).
  const ShapeCost& large = kShapes[0];
  const int64_t rounds = std::max<int64_t>(1, (t.k + 63) / 64), columns = t.after == After::kGated ? 2 * t.n : t.n;
  const int64_t across = (columns + large.n - 1) / large.n, down = (t.m + large.m - 1) / large.m, turns = across * down / large.at_once;
  if (turns == 0 || turns * large.at_once == across * down || t.after == After::kSlope) return best;  // (kSlope: 278 us and 279, a part of 4104 x 1000, 4096 inner)
  const int64_t rows = turns * large.at_once / across * large.m;
  if (rows == 0) return best;
  const double first = time_of(large, rows / large.m * across, rounds) + kLaunch;
  double least = best.time * 15 / 16;
  for (int shape = 1; shape < 4; ++shape) {
    if (!makes(shape, t.after)) continue;
    const ShapeCost& c = kShapes[shape];
    const double time = first + time_of(c, ((t.m - rows + c.m - 1) / c.m) * ((columns + c.n - 1) / c.n), rounds);
    if (time < least) {
      least = time;
      best = {{0, 1, (int)rounds * 64, (int)rows, shape}, time};
    }
  }
  return best;
}
LinearPlan plan_of(const Task& t) { return estimate(t).plan; }

// Two products of which neither needs the other, of one shape in one launch where that is faster.
struct TwoPlans {
  LinearPlan first, second;
  bool together;
};
TwoPlans plan_two(const Task* a, const Task* b) {  // null: not wanted
  TwoPlans best = {};
  const Estimate x = a ? estimate(*a) : Estimate{}, y = b ? estimate(*b) : Estimate{};
  best.first = x.plan;
  best.second = y.plan;
  if (!a || !b) return best;
  double least = x.time + y.time + kLaunch;
  for (int shape = 1; shape < 3; ++shape) {
    const ShapeCost& c = kShapes[shape];
    Shares p, q;
    shares_of(*a, c, p);
    shares_of(*b, c, q);
    for (int i = 0; i < p.n; ++i)
      for (int j = 0; j < q.n; ++j) {
        const int64_t groups = p.groups[i] + q.groups[j];
        const int64_t most = std::max(p.rounds[i], q.rounds[j]);
        // beyond one turn the compute units take one workgroup after another, the longer ones first
        const double in_turns = (double)(p.groups[i] * p.rounds[i] + q.groups[j] * q.rounds[j]) / c.at_once * c.full + ceil((double)groups / c.at_once) * c.once;
        const double time = p.joined[i] + q.joined[j] + (groups <= c.at_once ? time_of(c, groups, most) : std::max(most * c.full + c.once, 1.1 * in_turns));
        if (time < least) {
          least = time;
          best = {{shape, p.shares[i], (int)p.rounds[i] * 64}, {shape, q.shares[j], (int)q.rounds[j] * 64}, true};
        }
      }
  }
  return best;
}

int64_t sums_bytes(const LinearPlan& p, int64_t m, int64_t columns) { return p.shares > 1 ? m * columns * 4 * p.shares : 0; }

// Shares of the rows for the sums over them: one where there are few, else workgroups of 64 columns, at least 64 rows to each, some
// thousand in all.
int64_t row_shares(int64_t rows, int64_t columns) {
  if (rows <= kRowsAlone) return 1;
  const int64_t across = (columns + 63) / 64;
  return std::max<int64_t>(1, std::min<int64_t>({(rows + 63) / 64, std::max<int64_t>(1, 2048 / across), (int64_t)65535}));
}

// Those of a survey of dout, and its workgroups: some hundred, where each is to say what it found.
int64_t survey_shares(int64_t rows, int64_t columns, bool parts) {
  const int64_t across = (columns + kSlopeColumns - 1) / kSlopeColumns;
  return parts ? std::min(row_shares(rows, columns), std::max<int64_t>(1, 512 / across)) : row_shares(rows, columns);
}
int64_t survey_parts(int64_t rows, int64_t columns) { return survey_shares(rows, columns, true) * ((columns + kSlopeColumns - 1) / kSlopeColumns); }

// Places `first` .. `end` - 1 of rows of 16-bit values become 0, in blockIdx.y = 1 those `other` places behind them: a launch that only
// sizes which are no multiples of 8 cost, instead of comparisons in every tile (of which the largest spilled registers).
__global__ __launch_bounds__(256) void clear_places_kernel(uint16_t* matrix, int64_t rows, int64_t row, int32_t first, int32_t end, int32_t other) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= rows) return;
  for (int32_t i = first; i < end; ++i) matrix[r * row + blockIdx.y * (int64_t)other + i] = 0;
}

// ---- calls --------------------------------------------------------------------------------------------------------

struct Call {
  const char* what;
  bool bf16;
  hipStream_t stream;
  hipError_t error;
  Joins joins;
  uint32_t join_blocks;
  Call(const char* what_, int dtype, void* stream_)
      : what(what_), bf16(dtype == ND_BF16), stream((hipStream_t)stream_), error(hipSuccess), joins{}, join_blocks(0) {}
  void note(hipError_t e) {
    if (error == hipSuccess) error = e;
  }
  // A product of a forward pass, whose columns are rows of a matrix.
  void forward(const LinearParams& a, After after, float* sums) {
    if (a.m == 0) return;
    if (a.m <= kFewRows) {
      note(bf16 ? launch_few_rows<__bf16>(a, after, stream) : launch_few_rows<_Float16>(a, after, stream));
      return;
    }
    LinearParams p = a;
    p.sums = sums;
    // What the caches do not hold until the backward pass is written past them (8192 x 2 x 5632 at 3 bytes, 354 us and 351, and the product
    // behind it, which finds its operands there, 155 and 143; 3001 x 2 x 1000, both passes, 87 and 89), gated only where rows of its three parts begin with half lines: other pieces of 64 bytes are better put
    // together in the caches (both passes, 26020 x 2 x 456 175 us and 157, 8192 x 2 x 2728 594 and 562; 18436 x 2 x 1056 272 and 274, and
    // 30000 x 1000 without a gate 158 and 161).
    p.z_later = a.z && (int64_t)a.m * a.n * (after == After::kGated ? 6 : 2) > kCaches && (after != After::kGated || a.n % 32 == 0);
    const LinearPlan plan = plan_of({a.m, a.n, a.k, after});
    note(bf16 ? launch_linear<__bf16>(p, Layout::kRows, after, plan, stream) : launch_linear<_Float16>(p, Layout::kRows, after, plan, stream));
  }
  // What is to be added up at the end of the call.
  void join(const float* sums, int64_t shares, int64_t values, const float* factor, void* out) {
    Join& j = joins.job[joins.n++];
    j = {sums, out, factor, values / 8, (int32_t)shares, 1, join_blocks};
    // (few values: the reads of one lane follow each other)
    if (j.groups <= 1 << 14 && shares >= 4) j.lanes = shares >= 64 && j.groups <= 1 << 10 ? 32 : 8;
    join_blocks += (uint32_t)((j.groups * j.lanes + 255) / 256);
  }
  void add_up() {
    if (joins.n > 0) note(bf16 ? launch_joins<__bf16>(joins, join_blocks, stream) : launch_joins<_Float16>(joins, join_blocks, stream));
    joins.n = 0;
  }
  // One or two products of a backward pass (null: not wanted): by columns of the weights, and by columns.
  void backward(const LinearParams* a, After after, const LinearParams* b, const TwoPlans& plans) {
    if (a && a->m == 0) a = nullptr;
    if (plans.together && a && b) {
      note(bf16 ? launch_pair<__bf16>(*a, after, plans.first, *b, plans.second, stream) : launch_pair<_Float16>(*a, after, plans.first, *b, plans.second, stream));
    } else {
      if (a) one(*a, Layout::kWeightColumns, after, plans.first);
      if (b) one(*b, Layout::kColumns, After::kPlain, plans.second);
    }
    if (a && plans.first.shares > 1) join(a->sums, plans.first.shares, (int64_t)a->m * a->n, a->unscale, a->out);
    if (b && plans.second.shares > 1) join(b->sums, plans.second.shares, (int64_t)b->m * b->n, b->unscale, b->out);
  }
  void one(const LinearParams& a, Layout layout, After after, const LinearPlan& plan) {
    note(bf16 ? launch_linear<__bf16>(a, layout, after, plan, stream) : launch_linear<_Float16>(a, layout, after, plan, stream));
  }
  // dz and what is beside it; `total` gets the sums of the rows, unless it is null.
  void slope(const LinearParams& a, const void* dout, int64_t dout_bytes, float* sums, void* total, int64_t shares, float* parts) {
    float* parted = total && shares > 1 ? sums : nullptr;
    void* whole = shares > 1 ? nullptr : total;
    note(bf16 ? launch_slope<__bf16>(a, dout, dout_bytes, parted, whole, shares, parts, stream)
              : launch_slope<_Float16>(a, dout, dout_bytes, parted, whole, shares, parts, stream));
    if (parted) join(sums, shares, a.n, nullptr, total);
  }
  // The places of h or dz (gated: of both halves) that are filled up.
  void clear_filled(void* matrix, const nd_mlp* a, int halves) {
    if (a->inner_filled == 0 || a->rows == 0) return;
    clear_places_kernel<<<dim3((uint32_t)((a->rows + 255) / 256), halves), 256, 0, stream>>>((uint16_t*)matrix, a->rows, (int64_t)a->inner * halves,
                                                                                          a->inner - a->inner_filled, a->inner, a->inner);
    note(hipGetLastError());
  }
  // float16: dz made again where it leaves its range.
  void again(const LinearParams& a, const LinearPlan& plan) { note(launch_again<_Float16>(a, plan, stream)); }
  // Of dout [rows][columns]: the sums of its rows, unless out is null, and the largest of its values, unless parts is.
  void survey(const void* dout, int64_t row_bytes, int64_t rows, int32_t columns, float* sums, void* out, float* parts, uint32_t* found = nullptr) {
    LinearParams p = {};
    p.m = (int32_t)rows;
    p.n = columns;
    p.found = found;
    slope(p, dout, row_bytes, sums, out, survey_shares(rows, columns, parts), parts);
  }
  int done() const { return error == hipSuccess ? 0 : fail(std::string(what) + ": " + hipGetErrorString(error)); }
};

// dx [rows][dim] = dz weight;  dweight [out][dim] = dz^T x
LinearParams gradient_of_x(const void* dz, int64_t dz_bytes, const void* weight, int64_t rows, int32_t out, int32_t dim, float* unscale, void* dx, float* sums) {
  LinearParams p = {};
  p.p = weight;
  p.p_bytes = (int64_t)dim * 2;
  p.q = dz;
  p.q_bytes = dz_bytes;
  p.m = (int32_t)rows;
  p.n = dim;
  p.k = out;
  p.unscale = unscale;
  p.out = dx;
  p.sums = sums;
  return p;
}
LinearParams gradient_of_weight(const void* dz, int64_t dz_bytes, const void* x, int64_t x_bytes, int64_t rows, int32_t out, int32_t dim, float* unscale,
                                void* dweight, float* sums) {
  LinearParams p = {};
  p.p = x;
  p.p_bytes = x_bytes;
  p.q = dz;
  p.q_bytes = dz_bytes;
  p.m = out;
  p.n = dim;
  p.k = (int32_t)rows;
  p.unscale = unscale;
  p.out = dweight;
  p.sums = sums;
  return p;
}

std::string number(int64_t v) { return std::to_string(v); }

// Checks that both kinds of call share; an empty text if all is well.
std::string refuse(int64_t rows, std::initializer_list<int64_t> dims, int dtype, int activation, std::initializer_list<int64_t> strides) {
  if (dtype != ND_F16 && dtype != ND_BF16) return "16-bit types only (ND_F16, ND_BF16)";
  if (rows < 0 || rows > ND_LINEAR_MAX_ROWS) return "between 0 and " + number(ND_LINEAR_MAX_ROWS) + " rows, " + number(rows) + " given";
  for (const int64_t d : dims)
    if (d < 8 || d > ND_LINEAR_MAX_DIM || d % 8 != 0)
      return "sizes of vectors are multiples of 8 up to " + number(ND_LINEAR_MAX_DIM) + ", " + number(d) + " given";
  if (activation < ND_NO_ACTIVATION || activation > ND_SILU) return "unknown activation " + number(activation);
  for (const int64_t s : strides)
    if (s < 0 || s > ND_LINEAR_MAX_ROW_STRIDE || s % 8 != 0)
      return "rows lie a multiple of 8 elements apart, at most " + number(ND_LINEAR_MAX_ROW_STRIDE) + ", " + number(s) + " given";
  return "";
}

struct Array {
  const void* at;
  bool needed;
};
std::string refuse(std::initializer_list<Array> arrays) {
  for (const Array& a : arrays) {
    if (a.needed && !a.at) return "null array";
    if ((uintptr_t)a.at & 15) return "arrays are aligned to 16 bytes";
  }
  return "";
}

// Where the parts of a workspace lie.
struct Layouter {
  int64_t bytes = 0;
  int64_t take(int64_t n) {
    const int64_t at = bytes;
    bytes += round_up(n, 256);
    return at;
  }
};

int64_t forward_sums(int64_t m, int64_t n, int64_t k, bool gated) {
  return m <= kFewRows ? 0 : sums_bytes(plan_of({m, n, k, gated ? After::kGated : After::kForward}), m, gated ? 2 * n : n);
}

// ---- linear ---------------------------------------------------------------------------------------------------------

struct LinearWork {
  TwoPlans plans;  // dx, dweight
  int64_t dz, forward, dx, dweight, rows, parts, unscale, bytes;
};
LinearWork work_of(const nd_linear* a, bool backward) {
  LinearWork w = {};
  Layouter l;
  if (!backward) {
    w.forward = l.take(forward_sums(a->rows, a->out_dim, a->dim, false));
  } else {
    const bool active = a->activation != ND_NO_ACTIVATION, scaled = active && a->dtype == ND_F16;
    const Task dx = {a->rows, a->dim, a->out_dim, After::kPlain}, dweight = {a->out_dim, a->dim, a->rows, After::kPlain};
    w.plans = plan_two(a->dx ? &dx : nullptr, a->dweight ? &dweight : nullptr);
    w.dz = l.take(active ? a->rows * a->out_dim * 2 : 0);
    w.dx = l.take(a->dx ? sums_bytes(w.plans.first, dx.m, dx.n) : 0);
    w.dweight = l.take(a->dweight ? sums_bytes(w.plans.second, dweight.m, dweight.n) : 0);
    w.rows = l.take(a->dbias ? row_shares(a->rows, a->out_dim) * a->out_dim * 4 : 0);
    w.parts = l.take(scaled ? survey_parts(a->rows, a->out_dim) * 4 : 0);
    w.unscale = l.take(scaled ? 4 : 0);
  }
  w.bytes = l.bytes;
  return w;
}

std::string refuse(const nd_linear* a) {
  if (!a) return "null argument";
  return refuse(a->rows, {a->dim, a->out_dim}, a->dtype, a->activation, {a->x_row, a->residual_row, a->dout_row});
}

int run_linear(const nd_linear* a, bool backward, void* stream) {
  std::string why = refuse(a);
  if (!why.empty()) return fail("linear: " + why);
  const bool some = a->rows > 0, active = a->activation != ND_NO_ACTIVATION;
  if (!backward)
    why = refuse({{a->x, some}, {a->weight, some}, {a->bias, false}, {a->residual, false}, {a->out, some}, {a->z, false}});
  else
    why = refuse({{a->x, some && a->dweight}, {a->weight, some && a->dx}, {a->dout, some}, {a->z, some && active}, {a->dx, false}, {a->dweight, false}, {a->dbias, false}});
  if (!why.empty()) return fail("linear: " + why);
  const LinearWork w = work_of(a, backward);
  if (w.bytes > 0 && (a->workspace_bytes < w.bytes || !a->workspace || ((uintptr_t)a->workspace & 15)))
    return fail("linear: the workspace has " + number(a->workspace ? a->workspace_bytes : 0) + " bytes, " + number(w.bytes) + " needed, aligned to 16");
  char* work = (char*)a->workspace;
  Call call("linear", a->dtype, stream);
  if (!backward) {
    LinearParams p = {};
    p.p = a->weight;
    p.p_bytes = (int64_t)a->dim * 2;
    p.q = a->x;
    p.q_bytes = a->x_row * 2;
    p.m = (int32_t)a->rows;
    p.n = a->out_dim;
    p.k = a->dim;
    p.activation = a->activation;
    p.bias = a->bias;
    p.residual = a->residual;
    p.residual_bytes = a->residual_row * 2;
    p.out = a->out;
    p.z = a->z;
    call.forward(p, After::kForward, (float*)(work + w.forward));
    return call.done();
  }
  const void* dz = a->dout;
  int64_t dz_bytes = a->dout_row * 2;
  float *unscale = nullptr, *rows = (float*)(work + w.rows);
  if (active && (a->dx || a->dweight || a->dbias)) {
    LinearParams p = {};
    if (!call.bf16) {
      unscale = p.unscale = (float*)(work + w.unscale);
      p.parts = (const float*)(work + w.parts);
      p.n_parts = survey_parts(a->rows, a->out_dim);
      call.survey(a->dout, dz_bytes, a->rows, a->out_dim, nullptr, nullptr, (float*)(work + w.parts));
    }
    p.m = (int32_t)a->rows;
    p.n = a->out_dim;
    p.activation = a->activation;
    p.z = a->z;
    p.out = work + w.dz;
    call.slope(p, a->dout, dz_bytes, rows, a->dbias, row_shares(a->rows, a->out_dim), nullptr);
    dz = work + w.dz;
    dz_bytes = (int64_t)a->out_dim * 2;
  } else if (a->dbias) {
    call.survey(a->dout, dz_bytes, a->rows, a->out_dim, rows, a->dbias, nullptr);
  }
  const LinearParams dx = gradient_of_x(dz, dz_bytes, a->weight, a->rows, a->out_dim, a->dim, unscale, a->dx, (float*)(work + w.dx));
  const LinearParams dweight =
      gradient_of_weight(dz, dz_bytes, a->x, a->x_row * 2, a->rows, a->out_dim, a->dim, unscale, a->dweight, (float*)(work + w.dweight));
  call.backward(a->dx ? &dx : nullptr, After::kPlain, a->dweight ? &dweight : nullptr, w.plans);
  call.add_up();
  return call.done();
}

// ---- mlp --------------------------------------------------------------------------------------------------------------

struct MlpWork {
  TwoPlans first, second;  // dz and ddown; dx and dup
  int64_t shares;          // of the rows, whose sums the product that makes dz leaves
  int64_t dz, forward, dx, dup, ddown, rows, columns, parts, unscale, found, bytes;
};
MlpWork work_of(const nd_mlp* a, bool backward) {
  MlpWork w = {};
  Layouter l;
  const int64_t wide = (int64_t)a->inner * (a->gated ? 2 : 1);
  if (!backward) {
    w.forward = l.take(std::max(forward_sums(a->rows, a->inner, a->dim, a->gated), forward_sums(a->rows, a->out_dim, a->inner, false)));
  } else {
    const bool some = a->dx || a->dup || a->dup_bias, scaled = some && a->dtype == ND_F16;
    const Task dz = {a->rows, a->inner, a->out_dim, After::kSlope}, ddown = {a->out_dim, a->inner, a->rows, After::kPlain};
    const Task dx = {a->rows, a->dim, wide, After::kPlain}, dup = {wide, a->dim, a->rows, After::kPlain};
    w.first = plan_two(some ? &dz : nullptr, a->ddown ? &ddown : nullptr);
    w.second = plan_two(a->dx ? &dx : nullptr, a->dup ? &dup : nullptr);
    const int rows = kShapes[w.first.first.shape].m, waves[] = {Large::kWavesN, Medium::kWavesN, Small::kWavesN};
    w.shares = (a->rows + rows - 1) / rows * waves[std::min(w.first.first.shape, 2)];
    w.dz = l.take(some ? a->rows * wide * 2 : 0);
    w.dx = l.take(a->dx ? sums_bytes(w.second.first, dx.m, dx.n) : 0);
    w.dup = l.take(a->dup ? sums_bytes(w.second.second, dup.m, dup.n) : 0);
    w.ddown = l.take(a->ddown ? sums_bytes(w.first.second, ddown.m, ddown.n) : 0);
    w.rows = l.take(a->ddown_bias ? row_shares(a->rows, a->out_dim) * a->out_dim * 4 : 0);
    w.columns = l.take(a->dup_bias ? w.shares * wide * 4 : 0);
    w.parts = l.take(scaled ? survey_parts(a->rows, a->out_dim) * 4 : 0);
    w.unscale = l.take(scaled ? 4 : 0);
    w.found = l.take(scaled ? kExponents * 4 : 0);
  }
  w.bytes = l.bytes;
  return w;
}

std::string refuse(const nd_mlp* a) {
  if (!a) return "null argument";
  std::string why = refuse(a->rows, {a->dim, a->inner, a->out_dim}, a->dtype, a->activation, {a->x_row, a->residual_row, a->dout_row});
  if (why.empty() && a->gated && a->inner > ND_LINEAR_MAX_DIM / 2) why = "gated: at most " + number(ND_LINEAR_MAX_DIM / 2) + " inner places";
  if (why.empty() && (a->inner_filled < 0 || a->inner_filled >= a->inner))
    why = "between 0 and inner - 1 places are filled up, " + number(a->inner_filled) + " given";
  return why;
}

int run_mlp(const nd_mlp* a, bool backward, void* stream) {
  std::string why = refuse(a);
  if (!why.empty()) return fail("mlp: " + why);
  const bool some = a->rows > 0, first = a->dx || a->dup || a->dup_bias, slope = a->gated || a->activation != ND_NO_ACTIVATION;
  if (!backward)
    why = refuse({{a->x, some}, {a->up, some}, {a->down, some}, {a->up_bias, false}, {a->down_bias, false}, {a->residual, false}, {a->out, some}, {a->z, false}, {a->h, some}});
  else
    why = refuse({{a->x, some && a->dup}, {a->up, some && a->dx}, {a->down, some && first}, {a->z, some && first && slope}, {a->h, some && a->ddown},
                  {a->dout, some}, {a->dx, false}, {a->dup, false}, {a->dup_bias, false}, {a->ddown, false}, {a->ddown_bias, false}});
  if (!why.empty()) return fail("mlp: " + why);
  const MlpWork w = work_of(a, backward);
  if (w.bytes > 0 && (a->workspace_bytes < w.bytes || !a->workspace || ((uintptr_t)a->workspace & 15)))
    return fail("mlp: the workspace has " + number(a->workspace ? a->workspace_bytes : 0) + " bytes, " + number(w.bytes) + " needed, aligned to 16");
  char* work = (char*)a->workspace;
  Call call("mlp", a->dtype, stream);
  const int32_t wide = a->inner * (a->gated ? 2 : 1);
  const int64_t inner_bytes = (int64_t)a->inner * 2, wide_bytes = (int64_t)wide * 2;
  if (!backward) {
    LinearParams p = {};
    p.p = a->up;
    p.p_bytes = (int64_t)a->dim * 2;
    p.q = a->x;
    p.q_bytes = a->x_row * 2;
    p.m = (int32_t)a->rows;
    p.n = a->inner;
    p.k = a->dim;
    p.activation = a->activation;
    p.bias = a->up_bias;
    p.out = a->h;
    p.z = a->z;
    call.forward(p, a->gated ? After::kGated : After::kForward, (float*)(work + w.forward));
    call.clear_filled(a->h, a, 1);
    LinearParams r = {};
    r.p = a->down;
    r.p_bytes = inner_bytes;
    r.q = a->h;
    r.q_bytes = inner_bytes;
    r.m = (int32_t)a->rows;
    r.n = a->out_dim;
    r.k = a->inner;
    r.bias = a->down_bias;
    r.residual = a->residual;
    r.residual_bytes = a->residual_row * 2;
    r.out = a->out;
    call.forward(r, After::kForward, (float*)(work + w.forward));
    return call.done();
  }
  const int64_t dout_bytes = a->dout_row * 2;
  float* parts = first && some && !call.bf16 ? (float*)(work + w.parts) : nullptr;  // (without rows nobody leaves an unscale)
  float* unscale = parts ? (float*)(work + w.unscale) : nullptr;
  uint32_t* found = parts ? (uint32_t*)(work + w.found) : nullptr;
  if (a->ddown_bias || parts) call.survey(a->dout, dout_bytes, a->rows, a->out_dim, (float*)(work + w.rows), a->ddown_bias, parts, found);
  float* columns = a->dup_bias ? (float*)(work + w.columns) : nullptr;
  LinearParams p = {};
  p.p = a->down;
  p.p_bytes = inner_bytes;
  p.q = a->dout;
  p.q_bytes = dout_bytes;
  p.m = (int32_t)a->rows;
  p.n = a->inner;
  p.k = a->out_dim;
  p.activation = a->activation;
  p.gated = a->gated;
  p.z = slope ? a->z : nullptr;
  p.out = work + w.dz;
  p.parts = parts;
  p.n_parts = parts ? survey_parts(a->rows, a->out_dim) : 0;
  p.unscale = unscale;
  p.found = found;
  p.column_sums = columns;
  const LinearParams ddown =
      gradient_of_weight(a->dout, dout_bytes, a->h, inner_bytes, a->rows, a->out_dim, a->inner, nullptr, a->ddown, (float*)(work + w.ddown));
  call.backward(first ? &p : nullptr, After::kSlope, a->ddown ? &ddown : nullptr, w.first);
  if (parts) call.again(p, w.first.first);
  if (first) call.clear_filled(work + w.dz, a, a->gated ? 2 : 1);
  if (columns) call.join(columns, w.shares, wide, unscale, a->dup_bias);
  const char* dz = work + w.dz;
  const LinearParams dx = gradient_of_x(dz, wide_bytes, a->up, a->rows, wide, a->dim, unscale, a->dx, (float*)(work + w.dx));
  const LinearParams dup = gradient_of_weight(dz, wide_bytes, a->x, a->x_row * 2, a->rows, wide, a->dim, unscale, a->dup, (float*)(work + w.dup));
  call.backward(a->dx ? &dx : nullptr, After::kPlain, a->dup ? &dup : nullptr, w.second);
  call.add_up();
  return call.done();
}

}  // namespace
}  // namespace nd

extern "C" {

int64_t nd_linear_workspace(const nd_linear* a, int backward) {
  if (!nd::refuse(a).empty()) return -1;
  return nd::work_of(a, backward != 0).bytes;
}
int nd_linear_forward(const nd_linear* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_linear(a, false, stream); });
}
int nd_linear_backward(const nd_linear* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_linear(a, true, stream); });
}

int64_t nd_mlp_workspace(const nd_mlp* a, int backward) {
  if (!nd::refuse(a).empty()) return -1;
  return nd::work_of(a, backward != 0).bytes;
}
int nd_mlp_forward(const nd_mlp* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_mlp(a, false, stream); });
}
int nd_mlp_backward(const nd_mlp* a, void* stream) {
  return nd::guarded([&]() -> int { return nd::run_mlp(a, true, stream); });
}

}  // extern "C"
