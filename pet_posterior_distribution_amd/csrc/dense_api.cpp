// C-ABI implementation of the dense layer's operators (include/petdense.h): checks, the choice of tile and split for
// each product, and the launches.
#include "petdense.h"
#include "dense_internal.h"

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>

using namespace petdense_k;

namespace {

thread_local std::string g_err;

int fail(int code, const char* what) noexcept {
  try {
    g_err = what;
  } catch (...) {
  }
  return code;
}

#define HIPC(expr)                                                                         \
  do {                                                                                     \
    hipError_t e_ = (expr);                                                                \
    if (e_ != hipSuccess) return fail(PETDIFF_ERR_HIP, hipGetErrorString(e_));             \
  } while (0)
#define NEED(cond, what) \
  do {                   \
    if (!(cond)) return fail(PETDIFF_ERR_INVALID, what); \
  } while (0)

constexpr int64_t kMaxDim = 0x7fffffff - 0xffff;      // offsets a few steps and chunks past an end fit 31 bits
constexpr size_t kAlign = 256;

size_t up(size_t b) { return (b + kAlign - 1) / kAlign * kAlign; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int size_of(int dtype) { return dtype == PETDENSE_F32 ? 4 : 2; }

struct Plan {
  int tile = kSmall, splits = 1, c_per = 0;
  int b = 0, whole = 0;    // streamed products: rows of the tile, tiles that are not split
  bool stream = false;
  size_t part_bytes = 0;
  double us = 0;           // estimate
};

// What a kind of tile costs, in microseconds, as measured on products of 64 .. 12288 rows.  A step (128 bytes of
// contraction) takes `wait` when its workgroup has a compute unit to itself, and `share` per workgroup when several
// fill it; `ends` is a workgroup's first load and its epilogue.  [operands by DMA; through registers; dP formed there
// of ReLU or linear layers; of GELU and SiLU; one operand restored there from 8 bits]
struct Cost {
  int tile, b, slots, k;   // b: rows and columns of the tile; slots: workgroups of a compute unit; k: steps at a time
  double wait[5], share[5], ends;
};
constexpr int kFormed = 2, kFormedCurve = 3, kCodes = 4;
constexpr Cost kCosts16[] = {
    {kLarge, 256, 1, 1, {1.47, 0, 0, 0, 0}, {1.47, 0, 0, 0, 0}, 7.5},
    {kMid, 128, 2, 1, {0.65, 1.25, 0, 0, 0.95}, {0.46, 1.25, 0, 0, 0.62}, 3.5},
    {kSmall, 64, 4, 1, {0.28, 0.55, 2.0, 2.0, 0.65}, {0.19, 0.34, 1.5, 1.5, 0.3}, 2.0},
    {kSlice, 32, 1, 8, {0.5, 1.0, 1.8, 3.8, 0.65}, {1.2, 1.5, 3.0, 3.2, 1.4}, 2.0},
    {kSlice64, 64, 1, 4, {0.78, 2.4, 0, 0, 1.15}, {0.8, 2.4, 0, 0, 1.15}, 3.5}};
constexpr Cost kCosts32[] = {
    {kLarge, 256, 1, 1, {6.9, 0, 0, 0, 0}, {6.9, 0, 0, 0, 0}, 8.0},
    {kMid, 128, 2, 1, {2.3, 2.7, 0, 0, 2.5}, {2.1, 2.5, 0, 0, 2.3}, 4.0},
    {kSmall, 64, 4, 1, {0.75, 0.95, 2.4, 2.4, 0.87}, {0.53, 0.65, 2.0, 2.0, 0.6}, 2.0},
    {kSlice, 32, 1, 8, {1.1, 1.3, 1.9, 4.5, 1.3}, {1.3, 1.5, 3.5, 5.0, 1.5}, 2.0},
    {kSlice64, 64, 1, 4, {2.6, 4.5, 0, 0, 3.0}, {2.75, 4.5, 0, 0, 3.1}, 3.5}};
constexpr double kNever = 1e30;      // no plan
constexpr double kLaunch = 3.5;      // a launch behind another, here and on the host
constexpr double kWorkspace = 2.0;   // a small call that needs a workspace: the host's time for it
// The host's time for a call is longer than a small one's on the device: from Python 4 us forward, 8 us backward (its
// outputs), and 3.2 us a launch.  C callers and captured graphs spend less there and get the same plan: it goes by the
// arguments alone, so that a call has the same bits wherever it comes from.
constexpr double kHostForward = 4.0, kHostBackward = 8.0, kHostLaunch = 3.2;

// A call's price when calls follow each other: what is longer, the device's time or the host's (and a little for the
// device's where it is the host's, which a captured graph saves).
double call_us(double device, double host, int launches, bool work) {
  return std::max(device, host + kHostLaunch * launches + (work ? kWorkspace : 0.0)) + 0.02 * device;
}
constexpr int kUnits = 256;

double step_us(const Cost& c, double per_unit, int loader) {
  return std::max(c.wait[loader], c.share[loader] * per_unit);
}

// a workgroup's first load and its epilogue; through registers also its last step, whose pieces are cut to size
double ends_us(const Cost& c, int loader) { return c.ends + (loader == kReg ? 1.2 : 0.0); }

// `groups` workgroups of `steps` each, one after another where they are too many
double groups_us(const Cost& c, int64_t groups, int64_t steps, int loader) {
  const double per = (double)ceil_div(steps, c.k), ends = ends_us(c, loader);
  const int64_t whole = groups / (kUnits * c.slots), rest = groups % (kUnits * c.slots);
  double t = whole * (per * step_us(c, c.slots, loader) + ends);
  if (rest) {
    const double unit = rest < kUnits ? (double)rest / kUnits : (double)ceil_div(rest, kUnits);
    t += per * step_us(c, unit, loader) + ends;
  }
  return t;
}

double join_us(double values, int64_t splits) {
  return splits > 1 ? kLaunch + 1.0 + values * (splits + 1) * 4 / 3.5e6 : 0.0;
}

// Splits of `steps` into s <= most equal parts (the last may be shorter), few to many.
template <typename F>
void for_splits(int64_t steps, int64_t most, F f) {
  constexpr int kParts[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 56, 64};
  int64_t last = 0;
  for (const int want : kParts) {
    if (want > most || want > steps) break;
    const int64_t per = ceil_div(steps, want), s = ceil_div(steps, per);
    if (s == last) continue;
    last = s;
    f(s, per);
  }
}

// More parts than make twice the workgroups that the card holds gain nothing.
int64_t most_splits(const Cost& c, int64_t tiles) {
  return std::max<int64_t>(1, std::min<int64_t>(64, 2 * kUnits * c.slots / std::max<int64_t>(1, tiles)));
}

void set_plan(Plan& p, const Cost& c, int64_t splits, int64_t per, int bc, int64_t I, int64_t J) {
  p.tile = c.tile;
  p.splits = (int)splits;
  p.c_per = (int)std::min<int64_t>(per * bc, kMaxDim);
  p.part_bytes = splits > 1 ? up((size_t)splits * I * J * 4) : 0;
}

// operands read and outputs written once
double memory_us(double I, double J, double C, int type) {
  return (C * (I + J) + I * J) * (type == kF32 ? 4 : 2) / 4.5e6;
}

// Tile and split of a product by their estimated time; `call`: it is all of a call.
Plan plan(int64_t I, int64_t J, int64_t C, int type, int loader, bool call = false) {
  const int bc = type == kF32 ? 32 : 64;
  const int64_t steps = ceil_div(C, bc);
  const double memory = memory_us(I, J, C, type);
  Plan best;
  for (const Cost& c : type == kF32 ? kCosts32 : kCosts16) {
    if (c.tile == kLarge && loader != kDma) continue;
    const int64_t tiles = ceil_div(I, c.b) * ceil_div(J, c.b);
    if (c.k > 1 && tiles > 4 * kUnits) continue;        // sliced tiles are for few outputs
    const bool stream = c.tile == kLarge;
    // streamed: as many tiles whole as fill the card evenly, the others split; or all split
    const int64_t even = stream ? tiles / (kUnits * c.slots) * (kUnits * c.slots) : 0;
    for (int64_t whole : {(int64_t)0, even}) {
      const int64_t rest = tiles - whole;
      if (whole && !rest) continue;                    // nothing is left to split: the unsplit plan
      const double before = kLaunch + (whole ? groups_us(c, whole, steps, loader) : 0);
      if (best.c_per && before >= best.us) continue;
      for_splits(steps, whole ? 64 : most_splits(c, tiles), [&](int64_t s, int64_t per) {
        if (whole && s == 1) return;
        // split tiles' sums in fp32
        const double values = stream ? (double)rest * c.b * c.b : (double)I * J;
        if (s > 1 && values * s * 4 > 8e9) return;
        const double device =
            std::max(before + groups_us(c, rest * s, per, loader), kLaunch + 2.0 + memory) + join_us(values, s);
        const double t = call ? call_us(device, kHostForward, s > 1 ? 2 : 1, s > 1) : device;
        if (best.c_per && t >= best.us) return;
        best.us = t;
        set_plan(best, c, s, per, bc, I, J);
        best.stream = stream;
        best.b = c.b;
        best.whole = stream ? (int)(s > 1 ? whole : tiles) : 0;
        if (stream && s > 1) best.part_bytes = up((size_t)rest * c.b * c.b * s * 4);
      });
      if (!even) break;
    }
  }
  return best;
}

// The backward pass as one launch, or kNever where it has too many tiles for that: x (I = m, J = k, C = n) and k
// (I = k, J = n, C = m) with the same kind of tile; only the kernel gradient's contraction is split.  nx, nk: which
// products are wanted; `call`: it is all of a call (but for the join of a split).
double plan_pair(bool nx, bool nk, int64_t m, int64_t k, int64_t n, int type, int lx, int lk, bool slice64,
                 bool call, Plan& px, Plan& pk) {
  const int bc = type == kF32 ? 32 : 64;
  const int64_t sx = ceil_div(n, bc), sk = ceil_div(m, bc);
  const double memory = (nx ? memory_us(m, k, n, type) : 0) + (nk ? memory_us(k, n, m, type) : 0);
  double best = kNever, least = kNever;
  for (const Cost& c : type == kF32 ? kCosts32 : kCosts16) {
    if (c.tile == kLarge || c.tile == kMid || (c.tile == kSlice64 && !slice64)) continue;
    const int64_t tx = nx ? ceil_div(m, c.b) * ceil_div(k, c.b) : 0, tk = nk ? ceil_div(k, c.b) * ceil_div(n, c.b) : 0;
    if (tx > 16384 || tk > 16384) continue;
    if (c.k > 1 && tx + tk > 8 * kUnits) continue;
    for_splits(nk ? sk : 1, most_splits(c, tk), [&](int64_t s, int64_t per) {
      const double wx = nx ? (double)ceil_div(sx, c.k) : 0, wk = nk ? (double)ceil_div(nk ? per : 0, c.k) : 0;
      const double groups = (double)(tx + tk * s);
      const double ex = ends_us(c, lx), ek = ends_us(c, lk);
      const double share = ((double)tx * (wx * c.share[lx] + ex / c.slots) +
                            (double)tk * s * (wk * c.share[lk] + ek / c.slots)) / kUnits;
      const double longest = std::max(wx * c.wait[lx] + ex, wk * c.wait[lk] + ek);
      const double t = kLaunch + std::max({longest, share * (groups > kUnits * c.slots ? 1.25 : 1.0), 2.0 + memory}) +
                       (s > 1 ? join_us((double)k * n, s) + kWorkspace : 0.0);
      const double price = call ? call_us(t, kHostBackward, s > 1 ? 2 : 1, s > 1) : t;
      if (price >= least) return;
      least = price;
      best = t;
      set_plan(px, c, 1, sx, bc, m, k);
      set_plan(pk, c, s, per, bc, k, n);
      if (!nk) pk.splits = 1, pk.part_bytes = 0;
    });
  }
  return best;
}

// A whole product with a tile that is given.
double unsplit_us(int tile, int64_t I, int64_t J, int64_t C, int type, int loader) {
  const Cost& c = (type == kF32 ? kCosts32 : kCosts16)[tile];
  const int64_t tiles = ceil_div(I, c.b) * ceil_div(J, c.b), steps = ceil_div(C, type == kF32 ? 32 : 64);
  return kLaunch + std::max(groups_us(c, tiles, steps, loader), 2.0 + memory_us(I, J, C, type));
}

int64_t padded(int64_t n, int size) { return ceil_div(n, 16 / size) * (16 / size); }

// How an operand lies: DMA stages a whole tile's rows of it, or (free-contiguous) the rows of one step.
enum Lie { kAlongC, kAlongFree };

// These rows, `ld` values apart, lie within the 31-bit offsets that DMA has.
bool row_fits(int64_t ld, int size, Lie lie) {
  return ld < (lie == kAlongC ? kMaxRowBytes : 0x7fffffff / (128 / size)) / size;
}

bool dma_ok(const void* p, int64_t ld, int64_t contiguous, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row_fits(ld, size, kAlongC) && (ld * size) % 16 == 0 &&
         (contiguous * size) % 16 == 0;
}

bool planned(const Plan& p, int64_t C) {
  return p.c_per > 0 && (int64_t)p.splits * p.c_per >= C && (p.splits - 1) * (int64_t)p.c_per < C;
}

Product placed(Product p, const Plan& pl, void* part) {
  p.splits = pl.splits;
  p.c_per = pl.c_per;
  p.part = static_cast<float*>(part);
  p.whole = pl.whole;
  return p;
}

// `cols`: column sums that its join may carry (it has one where the plan splits)
int run_product(const Product& of, int layout, int loader, int type, int q8, const Plan& pl, void* part,
                const ColumnJoin& cols, hipStream_t s) {
  if (!planned(pl, of.C)) return fail(PETDIFF_ERR_HIP, "internal: a product without a plan");
  const Product p = placed(of, pl, part);
  HIPC(type == kF32    ? product_f32(p, layout, loader, pl.tile, q8, s)
       : type == kBF16 ? product_bf16(p, layout, loader, pl.tile, q8, s)
                       : product_f16(p, layout, loader, pl.tile, q8, s));
  if (pl.splits > 1) HIPC(pl.stream ? join_tiles(p, cols, type, pl.b, s) : join(p, cols, type, s));
  return PETDIFF_OK;
}

bool type_ok(int t) { return t >= PETDENSE_F32 && t <= PETDENSE_F16; }
bool act_ok(int a) { return a >= PETDENSE_NONE && a <= PETDENSE_SILU; }
bool work_ok(const void* w, size_t have, size_t need) {
  return need == 0 || (w && have >= need && reinterpret_cast<uintptr_t>(w) % kAlign == 0);
}

// No output that is given is an input or another output.
bool apart(std::initializer_list<const void*> outputs, std::initializer_list<const void*> inputs) {
  for (const void* const* o = outputs.begin(); o != outputs.end(); ++o) {
    if (!*o) continue;
    for (const void* i : inputs)
      if (*o == i) return false;
    for (const void* const* other = outputs.begin(); other != o; ++other)
      if (*o == *other) return false;
  }
  return true;
}

// a product's outputs: fewer than 2^23 tiles of 64 x 64
bool outputs_fit(int64_t i, int64_t j) { return ceil_div(i, 64) * ceil_div(j, 64) < (int64_t)1 << 23; }

// ---------------------------------------------------------------- forward
int check_forward(const petdense_forward_args* a) {
  NEED(a, "null arguments");
  NEED(type_ok(a->dtype), "dtype must be PETDENSE_F32, PETDENSE_BF16 or PETDENSE_F16");
  NEED(act_ok(a->activation), "unknown activation");
  NEED(a->m >= 0 && a->k >= 1 && a->n >= 1, "m must be >= 0, k and n >= 1");
  NEED(a->m < kMaxDim && a->k < kMaxDim && a->n < kMaxDim, "a dimension is too large");
  if (a->m == 0) return PETDIFF_OK;
  NEED(a->x && a->kernel && a->y, "x, kernel and y must be given");
  NEED(a->ldx >= a->k && a->ldk >= a->n && a->ldy >= a->n, "a row stride is shorter than its row");
  NEED(!a->residual || a->ldr >= a->n, "the residual's row stride is shorter than its row");
  NEED(!a->pre || a->ldp >= a->n, "the pre-activation's row stride is shorter than its row");
  NEED(apart({a->y, a->pre}, {a->x, a->kernel, a->bias}) && (!a->pre || a->pre != a->residual),
       "outputs must not alias inputs, nor each other");
  NEED(a->y != a->residual || (a->ldy == a->ldr && (!a->out_f32 || a->dtype == PETDENSE_F32)),
       "y may be the residual only with its stride and type");
  NEED(outputs_fit(a->m, a->n), "too many outputs in one call");
  return PETDIFF_OK;
}

// A copy of an operand that DMA can stage: its place in the workspace, or none.
struct Copy {
  bool on = false;
  size_t at = 0;
  int64_t ld = 0;
};

// Pieces of 16 bytes that the copy of an operand moves.  One launch copies fewer than kMaxPieces.
constexpr int64_t kMaxPieces = (int64_t)1 << 31;
int64_t pieces_of(bool on, int64_t rows, int64_t n, int size) { return on ? rows * (padded(n, size) * size / 16) : 0; }
// whether DMA can stage that copy
bool copy_fits(int64_t n, int size, Lie lie) { return row_fits(padded(n, size), size, lie); }
// read and written once, by a launch of its own
double copy_us(int64_t rows, int64_t n, int size) { return (double)rows * n * size * 2 / 3.5e6; }
constexpr double kCopyLaunch = kLaunch + 1.5;

Copy copy_of(bool on, int64_t rows, int64_t n, int size, size_t& o) {
  Copy c;
  if (!on) return c;
  c.on = true;
  c.at = o;
  c.ld = padded(n, size);
  o += up((size_t)rows * c.ld * size);
  return c;
}

PadJob job_of(const Copy& c, const void* src, int64_t ld, int64_t rows, int64_t n, char* w) {
  return c.on ? PadJob{src, w + c.at, ld, c.ld, (int)rows, (int)n} : PadJob{};
}

struct ForwardPlan {
  Plan p;
  int loader;
  bool rows;
  Copy x, kernel;
  size_t o_part, bytes;
};

ForwardPlan plan_forward(const petdense_forward_args* a) {
  ForwardPlan f{};
  f.rows = a->m <= kMaxRows && a->n <= 1 << 26;          // (a grid has fewer than 2^32 threads)
  if (a->m == 0) return f;
  if (f.rows) {
    // narrow layers leave compute units without columns: the contraction is split, where that is worth the join's
    // launch, 4 us and more of the host's (1 x 4096 x 1024: a call takes 8.0 us, 11.6 us split; rows that do not lie on
    // 16 bytes are slower: 1 x 3500 x 1356 takes 13.5 us on the device, 10.3 us split)
    const int64_t groups = ceil_div(a->n, kRowCols);
    const int64_t alone = dma_ok(a->kernel, a->ldk, a->n, size_of(a->dtype)) ? 5120 : 3584;
    const int64_t want = a->k >= alone ? std::min<int64_t>(kUnits / groups, a->k / 1024) : 1;
    f.p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, 16));
    f.p.c_per = (int)ceil_div(a->k, f.p.splits);
    f.p.splits = (int)ceil_div(a->k, f.p.c_per);
    f.bytes = f.p.splits > 1 ? up((size_t)f.p.splits * a->m * a->n * 4) : 0;
    return f;
  }
  const int sz = size_of(a->dtype);
  const bool x_ok = dma_ok(a->x, a->ldx, a->k, sz), w_ok = dma_ok(a->kernel, a->ldk, a->n, sz);
  f.loader = x_ok && w_ok ? kDma : kReg;
  f.p = plan(a->m, a->n, a->k, a->dtype, f.loader, true);
  size_t o = 0;
  if (f.loader == kReg) {
    const Plan q = plan(a->m, a->n, a->k, a->dtype, kDma, true);
    const double t = q.us + kCopyLaunch + (x_ok ? 0 : copy_us(a->m, a->k, sz)) + (w_ok ? 0 : copy_us(a->k, a->n, sz));
    // (x's rows are filled up with zeros; rows past the kernel's last are not read, which stages zeros too)
    if (t < f.p.us && (x_ok || copy_fits(a->k, sz, kAlongC)) && (w_ok || copy_fits(a->n, sz, kAlongFree)) &&
        pieces_of(!x_ok, a->m, a->k, sz) + pieces_of(!w_ok, a->k, a->n, sz) < kMaxPieces) {
      f.p = q;
      f.loader = kDma;
      f.x = copy_of(!x_ok, a->m, a->k, sz, o);
      f.kernel = copy_of(!w_ok, a->k, a->n, sz, o);
    }
  }
  f.o_part = o;
  f.bytes = o + f.p.part_bytes;
  return f;
}

// ---------------------------------------------------------------- backward
int check_backward(const petdense_backward_args* a) {
  NEED(a, "null arguments");
  NEED(type_ok(a->dtype), "dtype must be PETDENSE_F32, PETDENSE_BF16 or PETDENSE_F16");
  NEED(act_ok(a->activation), "unknown activation");
  NEED(a->m >= 0 && a->k >= 1 && a->n >= 1, "m must be >= 0, k and n >= 1");
  NEED(a->m < kMaxDim && a->k < kMaxDim && a->n < kMaxDim, "a dimension is too large");
  NEED(!a->dkernel || a->lddk >= a->n, "dkernel's row stride is shorter than its row");
  if (a->m > 0) {
    NEED(a->dy && a->lddy >= a->n, "dy must be given, with a row stride of at least n");
    NEED(a->activation == PETDENSE_NONE || (a->saved && a->lds >= a->n),
         "an activation's backward pass needs what the forward pass saved, with a row stride of at least n");
    NEED(!a->dx || (a->kernel && a->ldk >= a->n && a->lddx >= a->k),
         "dx needs the kernel, and row strides of the rows");
    NEED(!a->dkernel || (a->x && a->ldx >= a->k), "dkernel needs x, with a row stride of at least k");
    NEED(!a->dkernel || !a->x_exponents || a->lde >= ceil_div(a->k, PETDENSE_BLOCK),
         "the exponents' row stride is shorter than a row's blocks");
    NEED(!a->dresidual || a->lddr >= a->n, "dresidual's row stride is shorter than its row");
    NEED(apart({a->dx, a->dkernel, a->dbias, a->dresidual}, {a->dy, a->x, a->x_exponents, a->kernel, a->saved}),
         "outputs must not alias inputs, nor each other");
  }
  NEED((!a->dx || outputs_fit(a->m, a->k)) && (!a->dkernel || outputs_fit(a->k, a->n)),
       "too many outputs in one call");
  return PETDIFF_OK;
}

struct BackwardPlan {
  bool make_dp;            // dp is made by act_grad: in dresidual or in the workspace
  bool sums;               // column sums wanted
  bool fused;              // one launch for everything: dp is never in memory
  bool pair;               // one launch for both products and the bias gradient's join
  int chunks;
  Plan px, pk;
  int load_x, load_k;
  Copy dp, x, kernel;      // copies for DMA (dp: of dy or dresidual)
  bool restore;            // 8-bit inputs: x is their restored copy
  int64_t ld_dp;           // make_dp without dresidual: row stride of dp
  size_t o_dp, o_sums, o_part, bytes;
  double us;
};

// Column sums that a product's join may carry: 2^20 workgroups at most, in any of its grids.  More get a launch of
// their own, whose workgroups walk.
bool carried(int64_t n) { return n <= (int64_t)1 << 24; }

// The products from operands that are in memory (lx, lk: their loaders; dp_dma: dP's beside 8-bit inputs): one launch
// or two.
double plan_products(const petdense_backward_args* a, int lx, int lk, bool dp_dma, BackwardPlan& b) {
  const bool q8 = a->x_exponents;
  b.load_x = lx;
  b.load_k = lk;
  b.px = b.pk = Plan{};
  b.pair = false;
  if (a->dx) b.px = plan(a->m, a->k, a->n, a->dtype, lx);
  if (a->dkernel) b.pk = plan(a->k, a->n, a->m, a->dtype, lk);
  // a launch for the column sums, where no product's join carries them
  const bool joins =
      b.sums && !(carried(a->n) && ((a->dx && b.px.splits > 1) || (a->dkernel && b.pk.splits > 1)));
  double us = b.px.us + b.pk.us + (joins ? kLaunch : 0.0);
  if (a->dx && a->dkernel) {
    Plan px, pk;
    const double t = plan_pair(true, true, a->m, a->k, a->n, a->dtype, lx, lk, true, false, px, pk);
    if (t < us) {
      us = t;
      b.pair = true;
      b.px = px;
      b.pk = pk;
    }
  }
  // 8-bit inputs come through registers, or are restored into the workspace once where that costs less.  Their product
  // has a plan of its own; the input gradient keeps the tile and split that it has without them, and so its bits
  // (the price that is returned is the one without them: what it decides stays the same too).
  b.restore = false;
  if (q8 && a->dkernel) {
    const int sz = size_of(a->dtype);
    const double once = kCopyLaunch + (double)a->m * a->k * (1 + sz) / 3.5e6;
    const bool may = lk == kDma && copy_fits(a->k, sz, kAlongFree) && pieces_of(true, a->m, a->k, sz) < kMaxPieces;
    const Plan apart = plan(a->k, a->n, a->m, a->dtype, dp_dma ? kCodes : kReg);
    const Plan restored = plan(a->k, a->n, a->m, a->dtype, kDma);
    const bool cheaper = may && restored.us + once < apart.us;
    const double own = cheaper ? restored.us + once : apart.us;
    if (b.pair) {
      // the pair with the steps of a register load for the kernel's gradient, against launches of their own
      const double slower = us + (lk == kDma ? 1.25 * (apart.us - restored.us) : 0.0);
      const double alone = unsplit_us(b.px.tile, a->m, a->k, a->n, a->dtype, lx) + own + (joins ? kLaunch : 0.0);
      if (slower < alone) return us;
      b.pair = false;
    }
    b.pk = cheaper ? restored : apart;
    b.restore = cheaper;
  }
  return us;
}

BackwardPlan plan_backward(const petdense_backward_args* a) {
  BackwardPlan b{};
  const int sz = size_of(a->dtype);
  const bool q8 = a->x_exponents;
  b.make_dp = a->activation != PETDENSE_NONE || a->dresidual;
  b.sums = a->dbias != nullptr;
  const bool own_dp = b.make_dp && !a->dresidual;
  const int64_t ld_dp = ceil_div(a->n, 64) * 64;
  // row chunks of the activation's gradient: about 1024 workgroups, each of one round of its rows at least
  const int lanes = act_grad_lanes((int)a->n);
  const int64_t most = std::max<int64_t>(1, 1024 / ceil_div(a->n, lanes * 8));
  b.chunks = (int)std::max<int64_t>(1, std::min<int64_t>(most, ceil_div(a->m, 256 / lanes)));
  const double act_us =
      b.make_dp || b.sums ? kLaunch + 2.0 + (double)a->m * a->n * sz * (b.make_dp ? 3 : 1) / 4e6 : 0.0;

  // dp in the workspace has rows of whole pieces, with zeros: DMA takes it as it is.  dX's product reads dp and the
  // kernel along their contraction, dW's reads dp and x along their free values.
  const bool dp_ok =
      own_dp || (a->dresidual ? dma_ok(a->dresidual, a->lddr, a->n, sz) : dma_ok(a->dy, a->lddy, a->n, sz));
  const bool dp_x = !own_dp || row_fits(ld_dp, sz, kAlongC), dp_k = !own_dp || row_fits(ld_dp, sz, kAlongFree);
  const bool w_ok = !a->dx || dma_ok(a->kernel, a->ldk, a->n, sz);
  const bool x_ok = !a->dkernel || (q8 ? a->k * sz % 16 == 0 : dma_ok(a->x, a->ldx, a->k, sz));
  // (8-bit inputs go through registers whatever their alignment: their loader is dp's)
  b.us = act_us + plan_products(a, dp_ok && dp_x && w_ok ? kDma : kReg, dp_ok && dp_k && x_ok ? kDma : kReg,
                                dp_ok && dp_k, b);
  // with copies of what DMA does not take as it is, where their rows are short enough for it
  const bool copy_x = dp_x && (dp_ok || copy_fits(a->n, sz, kAlongC)) && (w_ok || copy_fits(a->n, sz, kAlongC));
  const bool copy_dp_k = dp_k && (dp_ok || copy_fits(a->n, sz, kAlongFree));
  const bool copy_k = copy_dp_k && (x_ok || q8 || copy_fits(a->k, sz, kAlongFree));
  const bool dp_on = !dp_ok && ((a->dx && copy_x) || (a->dkernel && copy_dp_k));
  const bool w_on = !w_ok && copy_x, x_on = !x_ok && !q8 && copy_k;
  if ((dp_on || w_on || x_on || (!x_ok && q8 && copy_k)) && (a->dx || a->dkernel) &&
      pieces_of(dp_on, a->m, a->n, sz) + pieces_of(w_on, a->k, a->n, sz) + pieces_of(x_on, a->m, a->k, sz) <
          kMaxPieces) {
    BackwardPlan c = b;
    c.us = act_us + plan_products(a, copy_x ? kDma : kReg, copy_k ? kDma : kReg, copy_dp_k, c) + kCopyLaunch +
           (dp_on ? copy_us(a->m, a->n, sz) : 0) + (w_on ? copy_us(a->k, a->n, sz) : 0) +
           (!x_ok && copy_k ? copy_us(a->m, a->k, sz) : 0);
    if (c.us < b.us) {
      b = c;
      b.dp.on = dp_on;
      b.kernel.on = w_on;
      b.x.on = x_on;
    }
  }
  // 8-bit inputs are staged through registers whatever their alignment: beside them dP takes the loader that it can
  if (q8 && a->dkernel && !b.restore && (b.dp.on ? copy_dp_k : dp_ok && dp_k)) b.load_k = kDma;
  // (dP is formed again for every tile that reads it: for small ones)
  if ((a->dx || a->dkernel) && (b.make_dp || b.sums) && !a->dresidual && a->m * a->n <= 1 << 18) {
    Plan px, pk;
    const int form = a->activation == PETDENSE_GELU || a->activation == PETDENSE_SILU ? kFormedCurve : kFormed;
    double t = plan_pair(a->dx, a->dkernel, a->m, a->k, a->n, a->dtype, form, form, false, true, px, pk);
    // a sum's workgroup walks all rows: 256 at a time, 4 of them in flight
    if (b.sums) t = std::max(t, kLaunch + 2.5 + 0.7 * (double)a->m / 256);
    const int joins = (a->dx && b.px.splits > 1 ? 1 : 0) + (a->dkernel && b.pk.splits > 1 ? 1 : 0);
    const int products = b.pair ? 1 : (a->dx ? 1 : 0) + (a->dkernel ? 1 : 0) + (b.sums && !joins ? 1 : 0);
    const int launches = 1 + products + joins + (b.dp.on || b.x.on || b.kernel.on ? 1 : 0);
    const bool split = a->dkernel && pk.splits > 1;
    if (call_us(t, kHostBackward, split ? 2 : 1, split) < call_us(b.us, kHostBackward, launches, true)) {
      b.us = t;
      b.fused = true;
      b.pair = false;
      b.px = px;
      b.pk = pk;
      b.dp.on = b.x.on = b.kernel.on = false;
    }
  }
  size_t o = 0;
  if (own_dp && !b.fused) {
    b.ld_dp = ld_dp;
    b.o_dp = o;
    o += up((size_t)a->m * b.ld_dp * sz);
  }
  if (b.sums && !b.fused) {
    b.o_sums = o;
    o += up((size_t)b.chunks * a->n * 4);
  }
  b.dp = copy_of(b.dp.on, a->m, a->n, sz, o);
  b.kernel = copy_of(b.kernel.on, a->k, a->n, sz, o);
  if (b.fused) b.restore = false;
  b.x = copy_of(b.x.on || b.restore, a->m, a->k, sz, o);
  b.o_part = o;
  b.bytes = o + std::max(b.px.part_bytes, b.pk.part_bytes);
  return b;
}

}  // namespace

extern "C" {

const char* petdense_last_error(void) { return g_err.c_str(); }

size_t petdense_forward_workspace(const petdense_forward_args* a) {
  if (check_forward(a) != PETDIFF_OK || a->m == 0) return 0;
  return plan_forward(a).bytes;
}

int petdense_forward(const petdense_forward_args* a, void* work, size_t work_bytes, void* stream) {
  if (int r = check_forward(a)) return r;
  if (a->m == 0) return PETDIFF_OK;
  const ForwardPlan f = plan_forward(a);
  NEED(work_ok(work, work_bytes, f.bytes), "the workspace is missing, too small or not 256-byte aligned");
  Product p{};
  p.A = a->x;
  p.lda = a->ldx;
  p.B = a->kernel;
  p.ldb = a->ldk;
  p.I = (int)a->m;
  p.J = (int)a->n;
  p.C = (int)a->k;
  p.e = Epilogue{a->bias, a->residual, a->y, a->pre, a->ldr, a->ldy, a->ldp, a->activation, a->bias_f32, a->out_f32};
  if (f.rows) {
    p = placed(p, f.p, work);
    HIPC(rows(p, a->dtype, (hipStream_t)stream));
    if (p.splits > 1) HIPC(join(p, ColumnJoin{}, a->dtype, (hipStream_t)stream));
    return PETDIFF_OK;
  }
  char* w = static_cast<char*>(work);
  if (f.x.on || f.kernel.on) {
    HIPC(pad(PadJobs{{job_of(f.x, a->x, a->ldx, a->m, a->k, w),
                      job_of(f.kernel, a->kernel, a->ldk, a->k, a->n, w), {}}},
             a->dtype, (hipStream_t)stream));
    if (f.x.on) p.A = w + f.x.at, p.lda = f.x.ld;
    if (f.kernel.on) p.B = w + f.kernel.at, p.ldb = f.kernel.ld;
  }
  return run_product(p, kForward, f.loader, a->dtype, 0, f.p, w + f.o_part, ColumnJoin{}, (hipStream_t)stream);
}

size_t petdense_backward_workspace(const petdense_backward_args* a) {
  if (check_backward(a) != PETDIFF_OK || a->m == 0) return 0;
  return plan_backward(a).bytes;
}

int petdense_backward(const petdense_backward_args* a, void* work, size_t work_bytes, void* stream) {
  if (int r = check_backward(a)) return r;
  hipStream_t s = (hipStream_t)stream;
  const int gsz = a->grad_f32 ? 4 : size_of(a->dtype);
  if (a->m == 0) {                                     // no rows: the sums over them are zero
    if (a->dkernel) HIPC(fill_zero(a->dkernel, a->k, a->n, a->lddk, gsz, s));
    if (a->dbias) HIPC(fill_zero(a->dbias, 1, a->n, a->n, gsz, s));
    return PETDIFF_OK;
  }
  const BackwardPlan b = plan_backward(a);
  NEED(work_ok(work, work_bytes, b.bytes), "the workspace is missing, too small or not 256-byte aligned");
  char* w = static_cast<char*>(work);
  float* sums = b.sums ? reinterpret_cast<float*>(w + b.o_sums) : nullptr;
  const void* dp = a->dy;
  int64_t lddp = a->lddy, n_dp = a->n;      // n_dp: dp's columns with the zeros behind them
  if (!b.fused && (b.make_dp || b.sums)) {
    void* made = nullptr;
    if (b.make_dp) {
      made = a->dresidual ? a->dresidual : w + b.o_dp;
      lddp = a->dresidual ? a->lddr : b.ld_dp;
      dp = made;
    }
    HIPC(act_grad(a->dy, a->lddy, a->activation == PETDENSE_NONE ? nullptr : a->saved, a->lds, made, lddp,
                  made && a->dresidual, sums, b.chunks, (int)a->m, (int)a->n, a->dtype, a->activation, s));
  }
  if (b.restore)
    HIPC(restore(static_cast<const uint8_t*>(a->x), a->ldx, a->x_exponents, a->lde, a->m, (int)a->k, a->dtype,
                 w + b.x.at, b.x.ld, s));
  if (b.dp.on || b.kernel.on || (b.x.on && !b.restore))
    HIPC(pad(PadJobs{{job_of(b.dp, dp, lddp, a->m, a->n, w), job_of(b.kernel, a->kernel, a->ldk, a->k, a->n, w),
                      b.restore ? PadJob{} : job_of(b.x, a->x, a->ldx, a->m, a->k, w)}},
             a->dtype, s));
  if (b.dp.on) dp = w + b.dp.at, lddp = b.dp.ld;
  if (b.load_x == kDma) n_dp = padded(a->n, size_of(a->dtype));
  const ColumnJoin cols{sums, a->dbias, b.chunks, b.sums ? (int)a->n : 0, a->grad_f32 ? kF32 : a->dtype};
  Product x{}, k{};
  if (a->dx) {
    x.A = dp;
    x.lda = lddp;
    x.B = b.kernel.on ? w + b.kernel.at : a->kernel;
    x.ldb = b.kernel.on ? b.kernel.ld : a->ldk;
    x.I = (int)a->m;
    x.J = (int)a->k;
    x.C = (int)n_dp;
    x.e.out = a->dx;
    x.e.ldo = a->lddx;
  }
  if (a->dkernel) {
    k.A = b.x.on ? w + b.x.at : a->x;
    k.lda = b.x.on ? b.x.ld : a->ldx;
    k.exps = b.restore ? nullptr : a->x_exponents;
    k.lde = a->lde;
    k.B = dp;
    k.ldb = lddp;
    k.I = (int)a->k;
    k.J = (int)a->n;
    k.C = (int)a->m;
    k.e.out = a->dkernel;
    k.e.ldo = a->lddk;
    k.e.out_f32 = a->grad_f32;
  }
  const int q8 = a->x_exponents != nullptr && !b.restore;
  if (b.fused || b.pair)
    if ((a->dx && !planned(b.px, a->n)) || (a->dkernel && !planned(b.pk, a->m)))
      return fail(PETDIFF_ERR_HIP, "internal: a product without a plan");
  if (b.fused) {
    const void* saved = a->activation == PETDENSE_NONE ? nullptr : a->saved;
    Pair p{};
    p.x = placed(x, b.px, nullptr);
    p.k = placed(k, b.pk, w + b.o_part);
    p.x.C = (int)a->n;
    p.x.A = p.k.B = a->dy;
    p.x.lda = p.k.ldb = a->lddy;
    p.x.saved = p.k.saved = saved;
    p.x.lds = p.k.lds = a->lds;
    p.x.saved_act = p.k.saved_act = a->activation;
    p.sums = ColumnSum{a->dy, saved, a->dbias, a->lddy, a->lds, (int)a->m, b.sums ? (int)a->n : 0, a->activation,
                       cols.out_type};
    HIPC(a->dtype == kF32    ? fused_f32(p, b.px.tile, q8, s)
         : a->dtype == kBF16 ? fused_bf16(p, b.px.tile, q8, s)
                             : fused_f16(p, b.px.tile, q8, s));
    if (a->dkernel && b.pk.splits > 1) HIPC(join(p.k, ColumnJoin{}, a->dtype, s));
    return PETDIFF_OK;
  }
  if (b.pair) {
    Pair p{};
    p.x = placed(x, b.px, nullptr);
    p.k = placed(k, b.pk, w + b.o_part);
    p.cols = cols;
    HIPC(a->dtype == kF32    ? pair_f32(p, b.load_x, b.load_k, b.px.tile, q8, s)
         : a->dtype == kBF16 ? pair_bf16(p, b.load_x, b.load_k, b.px.tile, q8, s)
                             : pair_f16(p, b.load_x, b.load_k, b.px.tile, q8, s));
    if (b.pk.splits > 1) HIPC(join(p.k, ColumnJoin{}, a->dtype, s));
    return PETDIFF_OK;
  }
  const bool with_x = carried(a->n) && a->dx && b.px.splits > 1;
  const bool with_k = carried(a->n) && !with_x && a->dkernel && b.pk.splits > 1;
  if (b.sums && !with_x && !with_k) HIPC(join_columns(cols, s));
  const ColumnJoin none{};
  char* part = w + b.o_part;
  if (a->dx)
    if (int r = run_product(x, kInputGrad, b.load_x, a->dtype, 0, b.px, part, with_x ? cols : none, s)) return r;
  if (a->dkernel)
    if (int r = run_product(k, kKernelGrad, b.load_k, a->dtype, q8, b.pk, part, with_k ? cols : none, s)) return r;
  return PETDIFF_OK;
}

int petdense_checkpoint(const void* x, int64_t ldx, int64_t m, int64_t k, int dtype, uint8_t* codes, int64_t ldc,
                        uint8_t* exponents, int64_t lde, void* stream) {
  NEED(type_ok(dtype), "dtype must be PETDENSE_F32, PETDENSE_BF16 or PETDENSE_F16");
  NEED(m >= 0 && k >= 1 && m < kMaxDim && k < kMaxDim, "m must be >= 0, k >= 1, both < 2^31 - 65536");
  if (m == 0) return PETDIFF_OK;
  NEED(x && codes && exponents, "x, codes and exponents must be given");
  NEED(ldx >= k && ldc >= k && lde >= ceil_div(k, PETDENSE_BLOCK), "a row stride is shorter than its row");
  NEED(apart({codes, exponents}, {x}), "outputs must not alias inputs, nor each other");
  HIPC(quantize(x, ldx, m, (int)k, dtype, codes, ldc, exponents, lde, (hipStream_t)stream));
  return PETDIFF_OK;
}

int petdense_restore(const uint8_t* codes, int64_t ldc, const uint8_t* exponents, int64_t lde, int64_t m, int64_t k,
                     int dtype, void* x, int64_t ldx, void* stream) {
  NEED(type_ok(dtype), "dtype must be PETDENSE_F32, PETDENSE_BF16 or PETDENSE_F16");
  NEED(m >= 0 && k >= 1 && m < kMaxDim && k < kMaxDim, "m must be >= 0, k >= 1, both < 2^31 - 65536");
  if (m == 0) return PETDIFF_OK;
  NEED(x && codes && exponents, "x, codes and exponents must be given");
  NEED(ldx >= k && ldc >= k && lde >= ceil_div(k, PETDENSE_BLOCK), "a row stride is shorter than its row");
  NEED(apart({x}, {codes, exponents}), "outputs must not alias inputs");
  HIPC(restore(codes, ldc, exponents, lde, m, (int)k, dtype, x, ldx, (hipStream_t)stream));
  return PETDIFF_OK;
}

}  // extern "C"
