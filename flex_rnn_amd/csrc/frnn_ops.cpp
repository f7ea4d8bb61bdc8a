// The operators linear_attention, linear_attention_step and layer_norm as PyTorch sees them: shapes and workspaces, argument
// blocks of the kernels in linear_attention.hip, layer_norm.hip and slice_sum.hip, their launches through the C ABI of
// frnn_rt.h, and their gradients.  One token of one user is a kernel of five microseconds: in Python its call took fifteen,
// and a gradient, which autograd runs on a thread of its own, a hundred.
//
// Code objects are built and loaded by flex_rnn_amd/handwritten.py, which this file asks for a kernel by number (`key` below)
// the first time that it needs one on a device.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/library.h>

#include <array>
#include <cstring>
#include <mutex>
#include <unordered_map>

#include "frnn_rt.h"

namespace {

using at::Tensor;
using std::optional;
typedef int64_t i64;

// ------------------------------------------------------------------ kernels
typedef i64 (*Loader)(i64 device, i64 key, char* message, i64 capacity);
Loader g_loader = nullptr;
std::mutex g_mutex;
std::unordered_map<i64, frnn_kernel_t> g_kernels;

// What a kernel is compiled for, in one number; the same fields as handwritten.py's `decode`.
enum Kind : i64 { BLOCK = 1, GATE = 2, STEP = 3, SUM = 4, NORM_FW = 5, NORM_BW = 6 };
i64 key_of(Kind kind, std::initializer_list<int> fields) {       // fields of 6 bits
  i64 k = kind;
  for (int f : fields) k = k << 6 | f;
  return k;
}

frnn_kernel_t kernel(i64 device, i64 key) {
  const i64 at = key << 8 | device;
  {
    std::lock_guard<std::mutex> lock(g_mutex);
    const auto it = g_kernels.find(at);
    if (it != g_kernels.end()) return it->second;
  }
  char message[4096] = "no loader";
  const i64 handle = g_loader ? g_loader(device, key, message, sizeof message) : 0;       // (not under the lock: it waits for Python)
  TORCH_CHECK(handle, message);
  std::lock_guard<std::mutex> lock(g_mutex);
  return g_kernels.emplace(at, (frnn_kernel_t)handle).first->second;
}

void launch(i64 device, i64 key, i64 grid_x, i64 grid_y, i64 threads, const void* args, size_t bytes) {
  if (grid_x <= 0 || grid_y <= 0) return;
  TORCH_CHECK(grid_x * threads < (1ll << 32), "a launch of ", grid_x, " workgroups is more than the hardware takes; split the batch");
  const uint32_t grid[3] = {(uint32_t)grid_x, (uint32_t)grid_y, 1}, block[3] = {(uint32_t)threads, 1, 1};
  const int rc = frnn_launch(kernel(device, key), grid, block, 0, (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(), args, bytes);
  TORCH_CHECK(rc == 0, "launching a kernel failed: ", frnn_last_error());
}

int type_of(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK(false, "bfloat16, float16 or float32 (got ", t, ")");
  }
}

i64 up(i64 a, i64 b) { return (a + b - 1) / b; }
void* ptr(const optional<Tensor>& t) { return t && t->defined() ? t->data_ptr() : nullptr; }

// ------------------------------------------------------------------ sums of slices
struct SumArgs {
  struct {
    const void* in;
    void* out;
  } pair[2];
  i64 S, X, type, cw, parts;
};

// out = the sum of S leading fp32 slices of in, for one or two pairs of one size and type
void slice_sums(i64 device, int n, const Tensor* in, const Tensor* out, i64 S) {
  const i64 X = out[0].numel();
  if (X == 0) return;
  // as many columns side by side (up to a 256-byte row of them) as leave 256 workgroups; the other threads share the slices
  i64 cw = 1;
  while (cw < 64 && cw < X && X / (2 * cw) * n >= 256) cw *= 2;
  // few slices of many columns: nothing to share, and 16-byte loads (2 x 4 M columns: 12 us against 74; 32 x 1 M: 22 and 25;
  // with more slices or fewer columns the two come out alike)
  if (S <= 32 && X % 4 == 0 && X >= 65536) cw = 1024;
  const i64 groups = up(X, cw);
  // many slices over few columns: parts of at least 16 trips per thread, joined by a second launch
  const i64 parts = cw > 256 ? 1 : std::max<i64>(1, std::min(512 / (groups * n), S / (16 * (256 / cw))));
  SumArgs a;
  for (int i = 0; i < 2; i++) a.pair[i] = {in[i % n].data_ptr(), out[i % n].data_ptr()};
  a.S = S, a.X = X, a.type = type_of(out[0].scalar_type()), a.cw = cw, a.parts = 1;
  Tensor part;
  if (parts > 1) {
    part = at::empty({n, parts, X}, in[0].options());
    SumArgs b = a;
    for (int i = 0; i < 2; i++) b.pair[i].out = (float*)part.data_ptr() + (i % n) * parts * X;
    b.type = 2, b.parts = parts;
    launch(device, key_of(SUM, {}), groups * parts, n, 256, &b, sizeof b);
    for (int i = 0; i < 2; i++) a.pair[i].in = b.pair[i].out;
    a.S = parts;
  }
  launch(device, key_of(SUM, {}), groups, n, 256, &a, sizeof a);
}

// ------------------------------------------------------------------ linear attention
constexpr i64 TOKENS = 32;            // per block
constexpr i64 UNITS = 256;            // compute units
constexpr i64 WORKGROUPS = 2 * UNITS; // below this a sequence is split into segments
constexpr i64 MAX_SEGMENTS = 64;

struct Operand {                      // struct Tensor of the kernels
  const void* p;
  i64 sb, st, sh, sn, vec;
};
struct Gate {
  const void* p;
  i64 sb, st, sh, type;
};
struct States {
  void* p;
  i64 sb, sh, sr, sc, type;
};
struct Job {
  Operand q, k, v, x;
  States init, fin;
  void* out;
  i64 ob, ot, og, os, share, out_type;
  void *dots, *marks, *inner, *local, *totals;
  i64 Hq, Hk, Hv, Hx, width, C, back, pairs;
  double in_scale, out_scale;
};
struct BlockArgs {
  Job job[2];
  Gate g;
  const void* lengths;
  i64 B, T, H, nseg, per, tiles, every;
};
struct GateArgs {
  const void *dots_q, *dots_k, *inner;
  Gate g;
  void* dg;
  const void* lengths;
  i64 B, T, H, tiles, type, init, every;
};
struct StepArgs {
  Operand q, k, v;
  Gate g;
  States s;
  void* y;
  i64 B, H, Hk, M, N, vec, gl, rows;
  double scale;
};

i64 width_of(i64 n) { return n <= 64 ? 64 : n <= 128 ? 128 : 256; }
int width_code(i64 w) { return w == 64 ? 0 : w == 128 ? 1 : 2; }

// Offsets within a block of tokens are 31 bits: a tensor whose block spans more is copied.
Tensor near(const Tensor& t) {
  return (TOKENS * t.stride(1) + 256 * t.stride(3)) * (i64)t.element_size() < (1ll << 31) ? t : t.contiguous();
}

Operand operand(const Tensor& t, bool time) {
  const i64 size = t.element_size(), st = time ? t.stride(1) : 0;
  Operand o = {t.data_ptr(), t.stride(0), st, t.stride(time ? 2 : 1), t.stride(-1), 0};
  if (o.sn == 1 && t.size(-1) >= 8) o.vec = t.size(-1) % 8 == 0 && ((i64)o.p | o.sb * size | o.st * size | o.sh * size) % 16 == 0 ? 1 : 2;
  return o;
}
Gate gate(const Tensor& g) {
  const i64 n = g.dim();
  return {g.data_ptr(), n > 1 ? g.stride(0) : 0, n > 2 ? g.stride(1) : 0, g.stride(-1), type_of(g.scalar_type())};
}
// [B,H,M,N] with rows N and columns M (as the walks that produce y and dv hold it), or rows M and columns N (dq, dk)
States states(const optional<Tensor>& s, bool rows_m) {
  if (!s || !s->defined()) return {nullptr, 0, 0, 0, 0, 2};
  return {s->data_ptr(), s->stride(0), s->stride(1), s->stride(rows_m ? 2 : 3), s->stride(rows_m ? 3 : 2), type_of(s->scalar_type())};
}

// (segments, blocks per segment) of a walk over `blocks` blocks by `groups` workgroups side by side.  Segments cost a second
// walk over k and v for the state at their starts, about half as long as the first, and a launch, about three blocks long:
// from 12 blocks on, segments of four and more win (T777, 24 workgroups: 53 us in two, 32 us in six).  Two workgroups per unit
// are worth up to 16 segments (T8192 H16 128x128: 97 us, 108 with one per unit); more, whose states each segment adds up, only
// reach for one (T16384 H4: 68 us in 32 segments, 84 in 64; T65536 H2: 91 in 64, 137 in 32).  All of these are bfloat16 or small
// heads, of which two workgroups fit a unit, and at most 64 walks: builds of which one fits (float16 over 128 columns, float32 over 64)
// and 65 to 511 walks go by the same rule unmeasured.
std::pair<i64, i64> segments(i64 groups, i64 blocks) {
  groups = std::max<i64>(groups, 1);
  const i64 n = std::min(std::max(std::min<i64>(up(WORKGROUPS, groups), 16), std::min(up(UNITS, groups), MAX_SEGMENTS)), blocks / 4);
  if (n <= 1 || blocks < 12) return {1, blocks};
  const i64 per = up(blocks, n);
  return {up(blocks, per), per};
}

// Borders at which the gradient of g starts anew, every 2^n blocks (see la_gate): at each for a decay that all tokens share, as long as
// the states that are written down there (a state of N rounded up to 16 by M rounded up to 64, 128 or 256, in fp32) take 8 GiB at most.
i64 every_of(i64 B, i64 T, i64 H, i64 M, i64 N, bool shared) {
  i64 n = shared ? 0 : 3;
  while (n < 3 && B * H * up(up(T, TOKENS), 1ll << n) > (1ll << 31) / (up(N, 16) * 16 * width_of(M))) n++;
  return n;
}

struct Problem {
  i64 device, B, T, H, Hk, M, N;
  int in;
  Gate g;
  i64 every;                          // of borders
  const void* lengths;
  at::TensorOptions bytes;            // float32 on the device: workspaces
};

Job job(const Problem& p, Operand q, i64 Hq, Operand k, i64 Hk, Operand v, i64 Hv, i64 width, i64 C, States init, States fin) {
  Job j;
  std::memset(&j, 0, sizeof j);
  j.q = q, j.k = k, j.v = v, j.init = init, j.fin = fin;
  j.x.vec = 1;
  j.Hq = Hq, j.Hk = Hk, j.Hv = Hv, j.Hx = 1;
  j.width = width, j.C = C, j.in_scale = j.out_scale = 1.0;
  return j;
}
// y or dv, [B,T,H,M]; dq or dk, [share][B,T,Hk,N]
void into(Job& j, const Problem& p, void* out, i64 heads, i64 n, i64 share, int type) {
  j.out = out, j.ob = p.T * heads * n, j.ot = heads * n, j.og = n, j.os = p.B * p.T * heads * n, j.share = share, j.out_type = type;
}

// One or two walks of one width and result type side by side, each in segments where the batch alone does not fill the chip.
void walk(const Problem& p, std::initializer_list<Job> jobs, bool dots) {
  BlockArgs a;
  std::memset(&a, 0, sizeof a);
  i64 n = 0;
  bool fast = true;
  for (const Job& j : jobs) {
    a.job[n++] = j;
    a.tiles = std::max(a.tiles, up(j.C, 64));
    fast = fast && j.C % 4 == 0 && j.q.vec == 1 && j.k.vec == 1 && j.v.vec == 1 && j.x.vec == 1;
  }
  const i64 w = width_of(a.job[0].width);
  a.g = p.g, a.lengths = p.lengths, a.B = p.B, a.T = p.T, a.H = p.H, a.every = p.every;
  std::tie(a.nseg, a.per) = segments(n * p.B * p.H * a.tiles, up(p.T, TOKENS));
  const int in = p.in, wc = width_code(w);
  Tensor local, totals;
  if (a.nseg > 1) {
    const i64 size = p.B * p.H * (a.nseg - 1);
    local = at::empty({n, size * a.tiles * 64 * w}, p.bytes);
    totals = at::empty({n, size}, p.bytes.dtype(at::kDouble));
    for (i64 i = 0; i < n; i++) {
      a.job[i].local = (float*)local.data_ptr() + i * local.size(1);
      a.job[i].totals = (double*)totals.data_ptr() + i * size;
    }
    launch(p.device, key_of(BLOCK, {in, wc, 0, 0, fast, 0}), up(size, 8) * 8 * a.tiles, n, 256, &a, sizeof a);
  }
  const bool wide = fast && a.job[0].out_type == 2 && in != 2;
  launch(p.device, key_of(BLOCK, {in, wc, 1, dots, fast, wide}), up(p.B * p.H * a.nseg, 8) * 8 * a.tiles, n, 256, &a, sizeof a);
}

// Offsets of results within a block of tokens are 31 bits, too.
constexpr i64 MAX_ROW = (1ll << 31) / (TOKENS * 4) - 1;

// What the kernels rely on; flex_rnn_amd/linear.py says what is wrong in words.
void check(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const optional<Tensor>& state, const optional<Tensor>& lengths, int lead) {
  const i64 B = q.size(0), Hk = q.size(-2), N = q.size(-1), H = v.size(-2), M = v.size(-1);
  bool ok = q.dim() == lead + 2 && q.sizes() == k.sizes() && v.dim() == lead + 2 && q.sizes().slice(0, lead) == v.sizes().slice(0, lead);
  ok = ok && Hk >= 1 && H >= 1 && H % Hk == 0 && N >= 1 && N <= 256 && M >= 1 && M <= 256 && (lead == 1 || (q.size(1) < (1ll << 31) - 64 && H * M <= MAX_ROW && Hk * N <= MAX_ROW));
  ok = ok && q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type();
  ok = ok && (g.dim() == 1 || (g.dim() == lead + 1 && g.sizes().slice(0, lead) == q.sizes().slice(0, lead))) && g.size(-1) == H;
  if (state) ok = ok && state->sizes() == at::IntArrayRef({B, H, M, N});
  if (lengths) ok = ok && lengths->dim() == 1 && lengths->size(0) == B && lengths->scalar_type() == at::kLong && lengths->is_contiguous();
  for (const Tensor* t : {&k, &v, &g}) ok = ok && t->device() == q.device();
  if (state) ok = ok && state->device() == q.device();
  if (lengths) ok = ok && lengths->device() == q.device();
  TORCH_CHECK(ok, "flex_rnn: shapes, types or devices of linear attention's operands do not go together");
}

Problem problem(const Tensor& q, const Tensor& v, const Tensor& g, const optional<Tensor>& lengths) {
  const Gate of_g = gate(g);
  return {q.device().index(), q.size(0), q.size(1), v.size(2), q.size(2), v.size(3), q.size(3), type_of(q.scalar_type()), of_g,
          every_of(q.size(0), q.size(1), v.size(2), v.size(3), q.size(3), of_g.st == 0),
          ptr(lengths), q.options().dtype(at::kFloat)};
}

Tensor state_like(const Tensor& v, i64 N, const optional<Tensor>& state) {
  return state ? at::empty_like(*state) : at::empty({v.size(0), v.size(2), v.size(3), N}, v.options().dtype(at::kFloat));
}

std::tuple<Tensor, Tensor> attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g, const optional<Tensor>& state,
                                     const optional<Tensor>& lengths, double scale) {
  check(q_, k_, v_, g, state, lengths, 2);
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = near(q_), k = near(k_), v = near(v_);
  const Problem p = problem(q, v, g, lengths);
  Tensor y = at::empty(v.sizes(), v.options()), out = state_like(v, p.N, state);
  Job j = job(p, operand(q, true), p.Hk, operand(k, true), p.Hk, operand(v, true), p.H, p.N, p.M, states(state, false), states(out, false));
  into(j, p, y.data_ptr(), p.H, p.M, 1, p.in);
  j.out_scale = scale;
  walk(p, {j}, false);
  return {y, out};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> attention_backward(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& g,
                                                                      const optional<Tensor>& state, const optional<Tensor>& lengths, const Tensor& dy_,
                                                                      const optional<Tensor>& dstate, double scale, bool need_g, bool need_state) {
  check(q_, k_, v_, g, state, lengths, 2);
  TORCH_CHECK(dy_.sizes() == v_.sizes() && dy_.scalar_type() == v_.scalar_type() && dy_.device() == v_.device(), "flex_rnn: dy is like y");
  if (dstate) TORCH_CHECK(dstate->sizes() == at::IntArrayRef({v_.size(0), v_.size(2), v_.size(3), q_.size(3)}) && dstate->device() == v_.device(), "flex_rnn: dstate is like the state");
  TORCH_CHECK(!need_state || state, "flex_rnn: no state to differentiate");
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = near(q_), k = near(k_), v = near(v_), dy = near(dy_);
  const Problem p = problem(q, v, g, lengths);
  const i64 share = p.H / p.Hk, tiles = up(p.N, 64), blocks = up(p.T, TOKENS), borders = up(blocks, 1ll << p.every) + 2;
  Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()), dv = at::empty(v.sizes(), v.options());
  Tensor ds = need_state ? at::empty_like(*state) : at::empty({0}, q.options()), dg;
  // heads that share a query and key each have their own share of its gradient
  Tensor part;
  void *pq = dq.data_ptr(), *pk = dk.data_ptr();
  if (share > 1) {
    part = at::empty({2, share, dq.numel()}, p.bytes);
    pq = part.data_ptr(), pk = (float*)pq + share * dq.numel();
  }
  const int type = share > 1 ? 2 : p.in;
  const Operand oq = operand(q, true), ok = operand(k, true), ov = operand(v, true), oy = operand(dy, true);
  const States none = states(optional<Tensor>(), true);
  Job of_q = job(p, oy, p.H, ov, p.H, ok, p.Hk, p.M, p.N, states(state, true), none);
  into(of_q, p, pq, p.Hk, p.N, share, type);
  of_q.out_scale = scale;
  Job of_k = job(p, ov, p.H, oy, p.H, oq, p.Hk, p.M, p.N, states(dstate, true), need_state ? states(ds, true) : none);
  into(of_k, p, pk, p.Hk, p.N, share, type);
  of_k.back = 1, of_k.in_scale = scale;
  Job of_v = job(p, ok, p.Hk, oq, p.Hk, oy, p.H, p.N, p.M, states(dstate, false), none);
  into(of_v, p, dv.data_ptr(), p.H, p.M, 1, p.in);
  of_v.back = 1, of_v.in_scale = scale;
  Tensor dots, marks, inner;
  if (need_g) {
    dots = at::empty({2, tiles, p.B * p.H, p.T}, p.bytes.dtype(at::kDouble));
    marks = at::empty({p.B * p.H * borders * up(p.N, 16) * 16 * width_of(p.M)}, p.bytes);
    inner = at::empty({p.B * p.H * borders, tiles * 4}, p.bytes.dtype(at::kDouble));
    for (Job* j : {&of_q, &of_k}) j->marks = marks.data_ptr(), j->inner = inner.data_ptr();
    of_q.pairs = 1, of_q.x = oq, of_q.Hx = p.Hk, of_q.dots = dots.data_ptr();
    of_k.x = ok, of_k.Hx = p.Hk, of_k.dots = (double*)dots.data_ptr() + dots.numel() / 2;
    // dq's walk multiplies with what dk's wrote down, so it comes later.  dv's goes along with dk's, at the price of dk's
    // three parts of the state, where one kernel serves both and the chip has room for them side by side (B2 T500 H8 64x48
    // fp32: 21 us less); by itself it takes two thirds of the time.
    const bool together = width_of(p.M) == width_of(p.N) && (share == 1 || p.in == 2) && 2 * p.B * p.H * std::max(tiles, up(p.M, 64)) <= WORKGROUPS;
    if (together) walk(p, {of_k, of_v}, true);
    else walk(p, {of_k}, true);
    walk(p, {of_q}, true);
    if (!together) walk(p, {of_v}, false);
  } else {
    walk(p, {of_q, of_k}, false);
    walk(p, {of_v}, false);
  }
  if (share > 1) {
    const Tensor in[2] = {part[0], part[1]}, out[2] = {dq, dk};
    slice_sums(p.device, 2, in, out, share);
  }
  if (need_g) {
    dg = at::empty(g.sizes(), g.options());
    const bool per_head = g.dim() == 1;
    const Tensor out = per_head ? at::empty({p.B, p.T, p.H}, p.bytes) : dg;
    const GateArgs a = {dots.data_ptr(), of_k.dots, inner.data_ptr(), p.g, out.data_ptr(), p.lengths, p.B, p.T, p.H, tiles, type_of(out.scalar_type()), state.has_value(), p.every};
    launch(p.device, key_of(GATE, {}), p.B * p.H * up(blocks, 32), 1, 1024, &a, sizeof a);
    if (per_head) slice_sums(p.device, 1, &out, &dg, p.B * p.T);
  } else {
    dg = at::empty({0}, g.options());
  }
  return {dq, dk, dv, dg, ds};
}

// Autograd finds that a tensor it has kept was written to.
void changed(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& state, double scale) {
  check(q, k, v, g, state, {}, 1);
  const c10::DeviceGuard guard(q.device());
  const i64 B = q.size(0), Hk = q.size(1), N = q.size(2), H = v.size(1), M = v.size(2), size = state.element_size(), ve = 16 / size;
  const int in = type_of(q.scalar_type());
  Tensor y = at::empty(v.sizes(), v.options());
  StepArgs a = {operand(q, false), operand(k, false), operand(v, false), gate(g), states(state, true), y.data_ptr(), B, H, Hk, M, N, 0, 1, 0, scale};
  a.vec = a.s.sc == 1 && N % ve == 0 && ((i64)a.s.p | a.s.sb * size | a.s.sh * size | a.s.sr * size) % 16 == 0;
  while (a.gl < 64 && a.gl * (a.vec ? ve : 1) < N) a.gl *= 2;
  // eight rows per lane, four in flight (128 sequences x 32 heads of 128x128: 111 us; with four rows 125, twelve 116, sixteen 112 but
  // 12 instead of 8 for four sequences)
  // and fewer where the batch does not give each SIMD two waves (one sequence x 32 heads: 5.8 us, 6.9 with eight)
  i64 each = 8;
  while (each > 1 && B * H * up(M, 64 / a.gl * each) < 2048) each /= 2;
  a.rows = std::min<i64>(M, 64 / a.gl * each);
  launch(q.device().index(), key_of(STEP, {in}), up(B * H * up(M, a.rows), 4), 1, 256, &a, sizeof a);
  changed(state);
  return y;
}

// ------------------------------------------------------------------ layer norm
constexpr i64 THREADS = 256 * 2 * 256;      // in flight: two workgroups of 256 per compute unit (measured on the forward pass over rows of 128, from one half to sixteen: 5.0 TB/s at two, 3.9 at eight; the backward pass and rows of a workgroup go by it, too)

struct NormArgs {
  const void *x, *dy;
  void* y;
  const void *w, *b;
  void *dw, *db;
  i64 rows, heads, C, sx, hx, sy, hy, w_type, b_type, vec, teams;
  double eps;
};

struct Shape {
  int wide, threads, pieces, lanes;         // pieces: of 16 bytes, per lane
};
// A row stays in the registers of up to 64 lanes with four pieces each; wider rows take a workgroup of 256, 512 or 1024 threads.
Shape shape_of(i64 C, i64 size) {
  const i64 pieces = up(C * size, 16);
  for (int k : {1, 2, 4})
    if (pieces <= 64 * k) {
      int lanes = 1;
      while (lanes * k < pieces) lanes *= 2;
      return {0, 256, k, lanes};
    }
  const int k = size == 4 ? 4 : 2;
  int threads = 256;
  while (threads * k < pieces) threads *= 2;
  return {1, threads, k, threads};
}

// as many rows side by side as keep the chip busy, a multiple of `heads` (a team of lanes keeps its head); of workgroups with 1024
// threads one per compute unit (128 of them: 54 us against 39 for 2048 rows of 16384 bfloat16; 512: 54)
i64 teams_of(i64 rows, i64 heads, i64 lanes) {
  return std::min(rows / heads, std::max<i64>(1, (lanes == 1024 ? 2 : 1) * THREADS / (lanes * heads))) * heads;
}

struct Rows {
  Tensor t;
  i64 outer, head;                          // strides
};
// The dimensions in front of the heads as one, copied only if they do not fold, or if a row's columns are apart.
Rows rows_of(const Tensor& x, bool per_head) {
  const i64 lead = x.dim() - (per_head ? 2 : 1);
  i64 outer = 0, below = -1;
  bool fold = x.stride(-1) == 1 || x.size(-1) == 1;
  for (i64 i = lead - 1; i >= 0 && fold; i--) {
    if (x.size(i) == 1) continue;
    if (below < 0) outer = x.stride(i);
    else fold = x.stride(i) == below;
    below = x.stride(i) * x.size(i);
  }
  if (!fold) return rows_of(x.contiguous(), per_head);
  return {x, outer, per_head ? x.stride(-2) : 0};
}

void check_norm(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b) {
  bool ok = x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384;
  for (const auto* p : {&w, &b})
    if (*p) {
      const Tensor& t = **p;
      ok = ok && (t.dim() == 1 || (t.dim() == 2 && x.dim() >= 2 && t.size(0) == x.size(-2))) && t.size(-1) == x.size(-1) && t.is_contiguous() && t.device() == x.device();
    }
  ok = ok && (!w || !b || w->sizes() == b->sizes());
  TORCH_CHECK(ok, "flex_rnn: shapes or devices of the norm's operands do not go together");
}

bool heads_apart(const optional<Tensor>& w, const optional<Tensor>& b) { return (w && w->dim() == 2) || (b && b->dim() == 2); }

void norm_launch(Kind kind, const Rows& x, const Rows& dy, const Tensor& out, const optional<Tensor>& w, const optional<Tensor>& b, void* dw, void* db,
                 i64 heads, i64 teams, double eps) {
  const i64 C = out.size(-1), size = out.element_size(), device = out.device().index();
  const Shape s = shape_of(C, size);
  NormArgs a = {x.t.data_ptr(), dy.t.defined() ? dy.t.data_ptr() : nullptr, out.data_ptr(), ptr(w), ptr(b), dw, db, out.numel() / C, heads, C,
                x.outer, x.head, dy.outer, dy.head, w ? type_of(w->scalar_type()) : 2, b ? type_of(b->scalar_type()) : 2, 0, teams, eps};
  a.vec = C * size >= 16;
  int lanes_log = 0;
  while (1 << lanes_log < s.lanes) lanes_log++;
  launch(device, key_of(kind, {type_of(out.scalar_type()), s.pieces, lanes_log, s.wide}), s.wide ? teams : up(teams * s.lanes, s.threads), 1,
         s.threads, &a, sizeof a);
}

Tensor norm(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps) {
  check_norm(x, w, b);
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return y;
  const bool per_head = heads_apart(w, b);
  const i64 heads = per_head ? x.size(-2) : 1, C = x.size(-1);
  norm_launch(NORM_FW, rows_of(x, per_head), {Tensor(), 0, 0}, y, w, b, nullptr, nullptr, heads,
              teams_of(x.numel() / C, heads, shape_of(C, x.element_size()).lanes), eps);
  return y;
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, const Tensor& dy, double eps, bool need_w,
                                                 bool need_b) {
  check_norm(x, w, b);
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(), "flex_rnn: dy is like y");
  TORCH_CHECK((!need_w || w) && (!need_b || b), "flex_rnn: no weight or bias to differentiate");
  const c10::DeviceGuard guard(x.device());
  Tensor dx = at::empty(x.sizes(), x.options());
  Tensor dw = need_w ? at::empty(w->sizes(), w->options()) : at::empty({0}, x.options()), db = need_b ? at::empty(b->sizes(), b->options()) : at::empty({0}, x.options());
  if (x.numel() == 0) {
    dw.zero_();
    db.zero_();
    return {dx, dw, db};
  }
  const bool per_head = heads_apart(w, b);
  const i64 heads = per_head ? x.size(-2) : 1, C = x.size(-1), teams = teams_of(x.numel() / C, heads, shape_of(C, x.element_size()).lanes);
  Tensor part;
  float *pw = nullptr, *pb = nullptr;
  if (need_w || need_b) {
    part = at::empty({need_w + need_b, teams * C}, x.options().dtype(at::kFloat));
    pw = need_w ? (float*)part.data_ptr() : nullptr;
    pb = need_b ? (float*)part.data_ptr() + need_w * teams * C : nullptr;
  }
  norm_launch(NORM_BW, rows_of(x, per_head), rows_of(dy, per_head), dx, w, {}, pw, pb, heads, teams, eps);
  if (need_w && need_b && dw.scalar_type() == db.scalar_type()) {
    const Tensor in[2] = {part[0], part[1]}, out[2] = {dw, db};
    slice_sums(x.device().index(), 2, in, out, teams / heads);
  } else {
    if (need_w) slice_sums(x.device().index(), 1, std::array<Tensor, 1>{part[0]}.data(), &dw, teams / heads);
    if (need_b) slice_sums(x.device().index(), 1, std::array<Tensor, 1>{part[need_w]}.data(), &db, teams / heads);
  }
  return {dx, dw, db};
}

// ------------------------------------------------------------------ shapes without data
std::tuple<Tensor, Tensor> attention_meta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const optional<Tensor>& state,
                                          const optional<Tensor>& lengths, double scale) {
  return {at::empty_symint(v.sym_sizes(), v.options()),
          state ? at::empty_like(*state) : at::empty_symint({v.sym_size(0), v.sym_size(2), v.sym_size(3), q.sym_size(3)}, v.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> attention_backward_meta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                                                           const optional<Tensor>& state, const optional<Tensor>& lengths, const Tensor& dy,
                                                                           const optional<Tensor>& dstate, double scale, bool need_g, bool need_state) {
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options()), at::empty_symint(v.sym_sizes(), v.options()),
          need_g ? at::empty_symint(g.sym_sizes(), g.options()) : at::empty({0}, g.options()), need_state ? at::empty_like(*state) : at::empty({0}, q.options())};
}
Tensor attention_step_meta(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& state, double scale) {
  changed(state);
  return at::empty_symint(v.sym_sizes(), v.options());
}
Tensor norm_meta(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps) { return at::empty_symint(x.sym_sizes(), x.options()); }
std::tuple<Tensor, Tensor, Tensor> norm_backward_meta(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, const Tensor& dy, double eps,
                                                      bool need_w, bool need_b) {
  return {at::empty_symint(x.sym_sizes(), x.options()), need_w ? at::empty_symint(w->sym_sizes(), w->options()) : at::empty({0}, x.options()),
          need_b ? at::empty_symint(b->sym_sizes(), b->options()) : at::empty({0}, x.options())};
}

// ------------------------------------------------------------------ gradients
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

template <class F>
const c10::TypedOperatorHandle<F> op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wanted(const optional<Tensor>& t) { return t && wanted(*t); }
optional<Tensor> maybe(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); }

// A result of a gradient: a gradient of that, in anything (`input` stands for all), is refused (it would silently miss terms).
struct Once : torch::autograd::Function<Once> {
  static Tensor forward(AutogradContext* ctx, const Tensor& result, const Tensor& input) { return result.view_as(result); }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(false, "linear_attention and layer_norm can be differentiated once");
  }
};
// A forward-mode derivative of an input would be lost without a word.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const optional<Tensor>& t) { return t && has_tangent(*t); }
template <class... Inputs>
void refuse_tangents(const char* what, const Inputs&... inputs) {
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !(has_tangent(inputs) || ...), what,
              " has no forward-mode derivative (an input has a tangent)");
}
// the first of `inputs` that asks for a gradient
Tensor asking(std::initializer_list<optional<Tensor>> inputs) {
  if (at::GradMode::is_enabled())
    for (const auto& t : inputs)
      if (wanted(t)) return *t;
  return Tensor();
}

bool captured(const c10::hip::HIPStream& s) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return s.stream() && hipStreamIsCapturing(s.stream(), &status) == hipSuccess && status == hipStreamCaptureStatusActive;
}
// In a backward pass that is being captured, a gradient for a node on the default stream - a leaf's, which belongs to the stream
// of an earlier graph that is still alive - makes autograd let that stream wait for the capture, which it cannot, on a thread
// where the error ends the process.  An error here does not.  (Any other stream joins the capture by waiting for it.)
void refuse_nodes_outside_capture(const Tensor& t) {
  if (!t.is_cuda() || !captured(c10::hip::getCurrentHIPStream(t.device().index()))) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto& e : node->next_edges()) {
    const auto s = e.is_valid() ? e.function->stream() : std::nullopt;
    TORCH_CHECK(!s || c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *s).stream(),
                "flex_rnn: a captured backward pass would make the default stream, a stream outside the capture, wait for it: an input has an autograd "
                "graph from before. Delete that graph's results first, or compute it on another stream");
  }
}

struct Attention : torch::autograd::Function<Attention> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const optional<Tensor>& state,
                               const optional<Tensor>& lengths, double scale) {
    at::AutoDispatchBelowAutograd below;
    static const auto call = op<decltype(attention)>("flex_rnn::linear_attention");
    auto [y, s] = call.call(q, k, v, g, state, lengths, scale);
    ctx->save_for_backward({q, k, v, g, state.value_or(Tensor()), lengths.value_or(Tensor())});
    ctx->saved_data["scale"] = scale;
    ctx->set_materialize_grads(false);
    return {y, s};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    variable_list out(7);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    refuse_nodes_outside_capture(s[0]);
    const Tensor dy = grads[0].defined() ? grads[0] : at::zeros_like(s[2], at::MemoryFormat::Contiguous);
    const bool need_state = s[4].defined() && ctx->needs_input_grad(4);
    static const auto call = op<decltype(attention_backward)>("flex_rnn::linear_attention_backward");
    auto [dq, dk, dv, dg, ds] =
        call.call(s[0], s[1], s[2], s[3], maybe(s[4]), maybe(s[5]), dy, maybe(grads[1]), ctx->saved_data["scale"].toDouble(), ctx->needs_input_grad(3), need_state);
    if (ctx->needs_input_grad(0)) out[0] = dq;
    if (ctx->needs_input_grad(1)) out[1] = dk;
    if (ctx->needs_input_grad(2)) out[2] = dv;
    if (ctx->needs_input_grad(3)) out[3] = dg;
    if (need_state) out[4] = ds;
    return out;
  }
};

std::tuple<Tensor, Tensor> attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const optional<Tensor>& state,
                                              const optional<Tensor>& lengths, double scale) {
  refuse_tangents("linear_attention", q, k, v, g, state);
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v) || wanted(g) || wanted(state))) {
    const auto r = Attention::apply(q, k, v, g, state, lengths, scale);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowAutograd below;
  static const auto call = op<decltype(attention)>("flex_rnn::linear_attention");
  return call.call(q, k, v, g, state, lengths, scale);
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> attention_backward_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g,
                                                                               const optional<Tensor>& state, const optional<Tensor>& lengths, const Tensor& dy,
                                                                               const optional<Tensor>& dstate, double scale, bool need_g, bool need_state) {
  refuse_tangents("linear_attention's gradient", q, k, v, g, state, dy, dstate);
  static const auto call = op<decltype(attention_backward)>("flex_rnn::linear_attention_backward");
  std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> r;
  {
    at::AutoDispatchBelowAutograd below;
    r = call.call(q, k, v, g, state, lengths, dy, dstate, scale, need_g, need_state);
  }
  const Tensor t = asking({q, k, v, g, state, dy, dstate});
  if (!t.defined()) return r;
  return {Once::apply(std::get<0>(r), t), Once::apply(std::get<1>(r), t), Once::apply(std::get<2>(r), t), Once::apply(std::get<3>(r), t), Once::apply(std::get<4>(r), t)};
}

Tensor attention_step_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& state, double scale) {
  refuse_tangents("linear_attention_step", q, k, v, g, state);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(wanted(q) || wanted(k) || wanted(v) || wanted(g) || wanted(state)), "linear_attention_step updates the state in place and cannot be differentiated");
  at::AutoDispatchBelowAutograd below;
  static const auto call = op<decltype(attention_step)>("flex_rnn::linear_attention_step");
  return call.call(q, k, v, g, state, scale);
}

struct Norm : torch::autograd::Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps) {
    at::AutoDispatchBelowAutograd below;
    static const auto call = op<decltype(norm)>("flex_rnn::layer_norm");
    ctx->save_for_backward({x, w.value_or(Tensor()), b.value_or(Tensor())});
    ctx->saved_data["eps"] = eps;
    return call.call(x, w, b, eps);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    refuse_nodes_outside_capture(s[0]);
    const bool need_w = s[1].defined() && ctx->needs_input_grad(1), need_b = s[2].defined() && ctx->needs_input_grad(s[1].defined() ? 2 : 1);
    static const auto call = op<decltype(norm_backward)>("flex_rnn::layer_norm_backward");
    auto [dx, dw, db] = call.call(s[0], maybe(s[1]), maybe(s[2]), grads[0], ctx->saved_data["eps"].toDouble(), need_w, need_b);
    variable_list out(4);
    if (ctx->needs_input_grad(0)) out[0] = dx;
    if (need_w) out[1] = dw;
    if (need_b) out[2] = db;
    return out;
  }
};

Tensor norm_autograd(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps) {
  refuse_tangents("layer_norm", x, w, b);
  if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b))) return Norm::apply(x, w, b, eps);
  at::AutoDispatchBelowAutograd below;
  static const auto call = op<decltype(norm)>("flex_rnn::layer_norm");
  return call.call(x, w, b, eps);
}

std::tuple<Tensor, Tensor, Tensor> norm_backward_autograd(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, const Tensor& dy, double eps,
                                                          bool need_w, bool need_b) {
  refuse_tangents("layer_norm's gradient", x, w, b, dy);
  static const auto call = op<decltype(norm_backward)>("flex_rnn::layer_norm_backward");
  std::tuple<Tensor, Tensor, Tensor> r;
  {
    at::AutoDispatchBelowAutograd below;
    r = call.call(x, w, b, dy, eps, need_w, need_b);
  }
  const Tensor t = asking({x, w, b, dy});
  if (!t.defined()) return r;
  return {Once::apply(std::get<0>(r), t), Once::apply(std::get<1>(r), t), Once::apply(std::get<2>(r), t)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(flex_rnn, m) {
  m.def("linear_attention(Tensor q, Tensor k, Tensor v, Tensor g, Tensor? state, Tensor? lengths, float scale) -> (Tensor, Tensor)");
  m.def(
      "linear_attention_backward(Tensor q, Tensor k, Tensor v, Tensor g, Tensor? state, Tensor? lengths, Tensor dy, Tensor? dstate, float scale, bool need_g, "
      "bool need_state) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor g, Tensor(a!) state, float scale) -> Tensor");
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_backward(Tensor x, Tensor? weight, Tensor? bias, Tensor dy, float eps, bool need_w, bool need_b) -> (Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(flex_rnn, CUDA, m) {
  m.impl("linear_attention", attention);
  m.impl("linear_attention_backward", attention_backward);
  m.impl("linear_attention_step", attention_step);
  m.impl("layer_norm", norm);
  m.impl("layer_norm_backward", norm_backward);
}
TORCH_LIBRARY_IMPL(flex_rnn, Meta, m) {
  m.impl("linear_attention", attention_meta);
  m.impl("linear_attention_backward", attention_backward_meta);
  m.impl("linear_attention_step", attention_step_meta);
  m.impl("layer_norm", norm_meta);
  m.impl("layer_norm_backward", norm_backward_meta);
}
TORCH_LIBRARY_IMPL(flex_rnn, Autograd, m) {
  m.impl("linear_attention", attention_autograd);
  m.impl("linear_attention_backward", attention_backward_autograd);
  m.impl("linear_attention_step", attention_step_autograd);
  m.impl("layer_norm", norm_autograd);
  m.impl("layer_norm_backward", norm_backward_autograd);
}

// For handwritten.py and the tests of the rules above.
extern "C" {
void frnn_ops_set_loader(Loader loader) { g_loader = loader; }
void frnn_ops_segments(i64 groups, i64 blocks, i64* out) { std::tie(out[0], out[1]) = segments(groups, blocks); }
i64 frnn_ops_every(i64 B, i64 T, i64 H, i64 M, i64 N, i64 shared) { return every_of(B, T, H, M, N, shared != 0); }
void frnn_ops_norm_shape(i64 rows, i64 heads, i64 C, i64 size, i64* out) {      // wide, threads, pieces, lanes, teams
  const Shape s = shape_of(C, size);
  out[0] = s.wide, out[1] = s.threads, out[2] = s.pieces, out[3] = s.lanes, out[4] = teams_of(rows, heads, s.lanes);
}
}
