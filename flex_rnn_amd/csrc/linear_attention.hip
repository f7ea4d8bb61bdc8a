// Linear attention with a decay for each head, in blocks of L tokens on the matrix cores (gfx950).
//
//     S_t = exp(g_t) S_(t-1) + v_t k_t^T,   y_t = scale * S_t q_t          S [M,N]; q, k [N]; v [M]
//
// With G_i the sum of g over the tokens of a block up to and including i, and S the state in front of the block,
//
//     y_i  = scale * ( exp(G_i) S q_i + sum_{j<=i} exp(G_i - G_j) (q_i.k_j) v_j )
//     S'   = exp(G_L) S + sum_j exp(G_L - G_j) v_j k_j^T
//
// so a block costs matrix products only, and the state is read and written once per L tokens.
//
// Compiled once per (IN, RP_, L, W..) by flex_rnn_amd/linear.py, which passes
//   IN    element type of q, k, v, dy: 0 bfloat16, 1 float16, 2 float32
//   WA    padded width (32, 64, 128 or 256) of the operand that every wave reads whole
//   WB    the same of the other operand (gradient kernel only)
//   L     tokens per block (32 or 64)
//   KERNEL_FW / KERNEL_WALK / KERNEL_GRAD / KERNEL_STEP: which kernel this code object holds
//
// Numbers on the matrix cores.  All products are v_mfma_f32_16x16x32_bf16: fp32 sums of bfloat16 factors.  A factor with
// more bits is a sum of RP bfloat16 parts (float16: 2, float32: 3; the parts hold every bit, because each takes the leading
// 8 bits of what is left), and a product of two such factors is the sum of the products of their parts, less those below the
// last bit that counts.  The bfloat16 exponent is that of float32, so nothing overflows on the way that would not in float32.
//   - factors read from memory are exact;
//   - the decayed products P = exp(G_i - G_j) q_i.k_j are rounded to RP parts (one rounding to the inputs' own precision,
//     2^-9 of the value on average below half a step, where y is rounded to the same type anyway);
//   - the decayed v (or k) that enters a state has three parts: the state is an fp32 result even where the inputs are not.
// The state itself stays in fp32 accumulators for the whole sequence.
//
// Layout.  Operand tiles sit in LDS as [token][column], one plane per part.  The matrix instruction's reduction index may be
// permuted as long as both factors use the same order; everything here uses the order of its own results - in a block of 32,
// lane group g = lane/16 holds {4g..4g+3, 16+4g..16+4g+3} - so an accumulator tile becomes an operand without leaving
// its registers (the state in y, checkpoints in the gradients), and ds_read_b64_tr_b16 delivers the same order for
// operands whose reduction index runs down a tile's rows.  Row strides: 4 (tiles read along rows) or 8 (tiles read
// down columns) dwords modulo 64, which spreads the 16 rows that a half wave touches over all 64 banks.
#include <hip/hip_runtime.h>

typedef unsigned int u32;
typedef unsigned short u16;
typedef unsigned long long u64;
typedef long long i64;
typedef __bf16 bh2 __attribute__((ext_vector_type(2)));
typedef __bf16 bh8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef u32 v2u __attribute__((ext_vector_type(2)));
typedef u32 v4u __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));

#define DEV static __device__ __forceinline__
#define DEV_MEMBER __device__ __forceinline__

#ifndef IN
#error "IN is not defined"
#endif

constexpr int ESZ = IN == 2 ? 4 : 2;          // bytes per element of q, k, v, dy
constexpr int RP = IN + 1;                    // bfloat16 parts of such an element
constexpr double LOG2E = 1.4426950408889634;
constexpr double NO_DECAY = -200.0;           // exp of less is zero in fp32; keeps the sums of logarithms finite

enum { BF16 = 0, FP16 = 1, FP32 = 2 };

struct Tensor {      // strides in elements; `vec`: 16-byte loads of 8 (4 of fp32) elements are allowed
  const char* p;
  i64 sb, st, sh, sn, vec;
};

struct States {      // [B,H,M,N] of a type, or p = null
  char* p;
  i64 sb, sh, sm, sn, type;
};

DEV float as_f(u32 x) { return __uint_as_float(x); }
DEV u32 as_u(float x) { return __float_as_uint(x); }
DEV float half_to_f(u16 h) { return (float)__builtin_bit_cast(_Float16, h); }

DEV u32 pack_rne(float a, float b) {           // two floats to bfloat16, to nearest even
  f2 v = {a, b};
  return __builtin_bit_cast(u32, __builtin_convertvector(v, bh2));
}
DEV u32 pack_top(float a, float b) { return __builtin_amdgcn_perm(as_u(b), as_u(a), 0x07060302u); }

// NP parts of the two floats a, b: parts [0, NP-1) by truncation (what is left is exact), the last one to nearest.
template <int NP>
DEV void split2(float a, float b, u32* out, int stride) {
  for (int i = 0; i < NP - 1; i++) {
    const float ta = as_f(as_u(a) & 0xffff0000u), tb = as_f(as_u(b) & 0xffff0000u);
    out[i * stride] = pack_top(a, b);
    a = a == ta ? 0.f : a - ta;                // (an infinity leaves nothing behind; a NaN stays one)
    b = b == tb ? 0.f : b - tb;
  }
  out[(NP - 1) * stride] = pack_rne(a, b);
}

template <int NP>
struct Frag {        // 8 elements of the reduction index per lane, NP parts
  v4u d[NP];
};

template <int NP>
DEV Frag<NP> make_frag(const float* x) {
  Frag<NP> f;
  u32 t[NP * 4];
  for (int i = 0; i < 4; i++) split2<NP>(x[2 * i], x[2 * i + 1], t + i, 4);
  for (int p = 0; p < NP; p++) f.d[p] = v4u{t[4 * p], t[4 * p + 1], t[4 * p + 2], t[4 * p + 3]};
  return f;
}

DEV void frag_floats(const v4u d, float* x) {
  for (int i = 0; i < 4; i++) {
    x[2 * i] = as_f(d[i] << 16);
    x[2 * i + 1] = as_f(d[i] & 0xffff0000u);
  }
}

template <int NP>
DEV void frag_values(const Frag<NP>& f, float* x) {
  frag_floats(f.d[NP - 1], x);
  for (int p = NP - 2; p >= 0; p--) {
    float t[8];
    frag_floats(f.d[p], t);
    for (int i = 0; i < 8; i++) x[i] += t[i];
  }
}

// c += a b, the products of parts i, j with i + j <= LIM, smallest first
template <int LIM, int PA, int PB>
DEV f4 mul(const Frag<PA>& a, const Frag<PB>& b, f4 c) {
#pragma unroll
  for (int s = LIM; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < PA; i++) {
      const int j = s - i;
      if (j >= 0 && j < PB)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bh8, a.d[i]), __builtin_bit_cast(bh8, b.d[j]), c, 0, 0, 0);
    }
  return c;
}
constexpr int RAW = RP == 1 ? 0 : 2;           // both factors exact
constexpr int CALC = RP - 1;                   // one factor rounded to RP parts

// ------------------------------------------------------------------ LDS tiles
constexpr int stride_down(int w) { return w + 16; }       // for tiles read down their columns
constexpr int stride_along(int w) { return w + 8; }

DEV v4s tr_read(const u16* p) {
  typedef __attribute__((address_space(3))) v4s* lds_ptr;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(__attribute__((address_space(3))) void*)p);
}

// lane (p = lane % 16, g = lane / 16) gets column c0 + p, rows r0 + {4g..4g+3, 16+4g..16+4g+3}
template <int STR, int ROWS>
DEV Frag<RP> down(const u16* tile, int r0, int c0, int lane) {
  const int p = lane & 15, g = lane >> 4;
  const u16* at = tile + (r0 + 4 * g + (p >> 2)) * STR + c0 + 4 * (p & 3);
  Frag<RP> f;
#pragma unroll
  for (int i = 0; i < RP; i++) {
    const v2u a = __builtin_bit_cast(v2u, tr_read(at + i * ROWS * STR));
    const v2u b = __builtin_bit_cast(v2u, tr_read(at + i * ROWS * STR + 16 * STR));
    f.d[i] = v4u{a[0], a[1], b[0], b[1]};
  }
  return f;
}

// lane (p, g) gets row r, columns c0 + {4g..4g+3, 16+4g..16+4g+3}
template <int STR, int ROWS>
DEV Frag<RP> along(const u16* tile, int r, int c0, int g) {
  const u16* at = tile + r * STR + c0 + 4 * g;
  Frag<RP> f;
#pragma unroll
  for (int i = 0; i < RP; i++) {
    const v2u a = *(const v2u*)(at + i * ROWS * STR), b = *(const v2u*)(at + i * ROWS * STR + 16);
    f.d[i] = v4u{a[0], a[1], b[0], b[1]};
  }
  return f;
}

// lane (p, g) gets row r, columns c0 + 8g..8g+7: where the order is free on both sides
template <int STR, int ROWS>
DEV Frag<RP> along8(const u16* tile, int r, int c0, int g) {
  Frag<RP> f;
#pragma unroll
  for (int i = 0; i < RP; i++) f.d[i] = *(const v4u*)(tile + i * ROWS * STR + r * STR + c0 + 8 * g);
  return f;
}

// ------------------------------------------------------------------ memory to registers
struct Raw {         // 8 elements as they are in memory
  v4u d[ESZ / 2];
};

// `base`: the first token of the block (wave uniform); tokens from `rows` on and columns from `cols` on are zero.  Whether
// memory is read is decided before the address is formed: nothing outside the tensor is touched.
DEV Raw load8(const char* base, i64 st, i64 sn, bool vec, int row, int col, int rows, int cols) {
  Raw r;
  if (vec) {
    const bool ok = row < rows && col < cols;               // (cols is a multiple of 8 here)
    const v4u* at = (const v4u*)(base + (row * st + col) * ESZ);
    for (int i = 0; i < ESZ / 2; i++) r.d[i] = ok ? at[i] : v4u{0, 0, 0, 0};
  } else {
    u32 w[8];
    for (int e = 0; e < 8; e++) {
      const bool ok = row < rows && col + e < cols;
      const char* at = base + (row * st + (col + e) * sn) * ESZ;
      if constexpr (ESZ == 4) w[e] = ok ? *(const u32*)at : 0u;
      else w[e] = ok ? *(const u16*)at : 0u;
    }
    if constexpr (ESZ == 4) {
      r.d[0] = v4u{w[0], w[1], w[2], w[3]};
      r.d[ESZ / 2 - 1] = v4u{w[4], w[5], w[6], w[7]};
    } else {
      r.d[0] = v4u{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
    }
  }
  return r;
}

template <int PLANE>
DEV void store_parts(u16* at, const Raw& r) {
  if constexpr (IN == BF16) {
    *(v4u*)at = r.d[0];
  } else {
    float x[8];
    for (int e = 0; e < 8; e++) {
      if constexpr (IN == FP16) x[e] = half_to_f((u16)(r.d[0][e / 2] >> (e % 2 * 16)));
      else x[e] = as_f(r.d[e / 4][e % 4]);
    }
    const Frag<RP> f = make_frag<RP>(x);
    for (int p = 0; p < RP; p++) *(v4u*)(at + p * PLANE) = f.d[p];
  }
}

// a tile of ROWS tokens x W columns, staged by THREADS threads
template <int W, int STR, int ROWS, int THREADS>
struct Staging {
  static constexpr int UNITS = ROWS * (W / 8);
  static constexpr int N = (UNITS + THREADS - 1) / THREADS;
  Raw r[N];

  DEV_MEMBER void load(const char* base, const Tensor& t, int rows, int cols, int tid) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int u = tid + i * THREADS;
      if (UNITS % THREADS == 0 || u < UNITS) r[i] = load8(base, t.st, t.sn, t.vec != 0, u / (W / 8), u % (W / 8) * 8, rows, cols);
    }
  }
  DEV_MEMBER void store(u16* tile, int tid) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int u = tid + i * THREADS;
      if (UNITS % THREADS == 0 || u < UNITS) store_parts<ROWS * STR>(tile + u / (W / 8) * STR + u % (W / 8) * 8, r[i]);
    }
  }
};

DEV float load_type(const char* p, i64 i, int type) {
  if (type == FP32) return ((const float*)p)[i];
  const u16 h = ((const u16*)p)[i];
  return type == FP16 ? half_to_f(h) : as_f((u32)h << 16);
}
DEV void store_type(char* p, i64 i, int type, float x) {
  if (type == FP32) ((float*)p)[i] = x;
  else if (type == FP16) ((_Float16*)p)[i] = (_Float16)x;
  else ((u16*)p)[i] = (u16)pack_rne(x, 0.f);
}

// ------------------------------------------------------------------ decays of a block
template <int CTRL, int ROW_MASK>
DEV double dpp_or_zero(double x) {
  const u64 b = __builtin_bit_cast(u64, x);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROW_MASK, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROW_MASK, 0xf, false);
  return __builtin_bit_cast(double, (u64)(u32)hi << 32 | (u32)lo);
}
DEV double scan64(double x) {                  // inclusive sums over the 64 lanes
  x += dpp_or_zero<0x111, 0xf>(x);             // row_shr 1, 2, 4, 8: within rows of 16
  x += dpp_or_zero<0x112, 0xf>(x);
  x += dpp_or_zero<0x114, 0xf>(x);
  x += dpp_or_zero<0x118, 0xf>(x);
  x += dpp_or_zero<0x142, 0xa>(x);             // a row's last lane into the next row
  x += dpp_or_zero<0x143, 0xc>(x);             // lane 31 into the upper half
  return x;
}
DEV double last_lane(double x) {
  const u64 b = __builtin_bit_cast(u64, x);
  const u32 lo = __builtin_amdgcn_readlane((int)b, 63), hi = __builtin_amdgcn_readlane((int)(b >> 32), 63);
  return __builtin_bit_cast(double, (u64)hi << 32 | lo);
}

struct Gate {        // g: [B,T,H] (or [H]: strides 0)
  const char* p;
  i64 sb, st, sh, type;
};

DEV double gate_of(const Gate& g, i64 b, i64 h, i64 t) {
  const double x = load_type(g.p, b * g.sb + t * g.st + h * g.sh, (int)g.type);
  return x < NO_DECAY ? NO_DECAY : x;
}

template <int L_>
struct Decays {
  // G * log2(e) as a sum of two floats: differences of far sums keep the precision of near ones
  float hi[L_], lo[L_];
  float from_start[L_], to_end[L_];            // exp(G_i), exp(G_L - G_i)
  float all;                                   // exp(G_L)
};

// one wave; lane i holds token i's g (0 behind the last token)
template <int L_>
DEV double fill_decays(Decays<L_>& d, double g, int lane) {
  const double G = scan64(g), end = last_lane(G);
  if (lane < L_) {
    const double G2 = G * LOG2E;
    const float hi = (float)G2;
    d.hi[lane] = hi;
    d.lo[lane] = (float)(G2 - (double)hi);
    d.from_start[lane] = expf((float)G);
    d.to_end[lane] = expf((float)(end - G));
    if (lane == 0) d.all = expf((float)end);
  }
  return end;
}

template <int L_>
DEV float decay_between(const Decays<L_>& d, float hi_i, float lo_i, int j) {
  return __builtin_amdgcn_exp2f((hi_i - d.hi[j]) + (lo_i - d.lo[j]));
}

// Workgroups go to the 8 XCDs in turn; the `n` workgroups of one group (which read the same operands) get numbers 8 apart
// and so share an L2.
DEV bool spread(u32 id, int n, i64 groups, i64* group, int* member) {
  const u32 x = id & 7, y = id >> 3;
  *group = (i64)(y / (u32)n) * 8 + x;
  *member = (int)(y % (u32)n);
  return *group < groups;
}

DEV i64 length_of(const i64* lengths, i64 b, i64 T) {
  if (!lengths) return T;
  const i64 n = lengths[b];
  return n < 0 ? 0 : n > T ? T : n;
}

DEV void tile_of(int idx, int* it, int* jt) {   // the idx-th tile on or below the diagonal, row by row
  const int i = (idx >= 1) + (idx >= 3) + (idx >= 6);
  *it = i;
  *jt = idx - i * (i + 1) / 2;
}

DEV float sum16(float x) {                     // over the 16 lanes of a row
  for (int m = 1; m < 16; m <<= 1) x += __shfl_xor(x, m, 64);
  return x;
}
DEV float sum_groups(float x) {                // over the 4 lanes with the same lane % 16
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// ================================================================== forward pass
#ifdef KERNEL_FW
// One workgroup walks the blocks of one (batch, head, segment) for 64 of the M columns of v; wave w owns 16 of them: its
// share of the state, S^T [WA x 16], stays in accumulators.  q and k are read by every workgroup of a head (up to four,
// on one XCD).  The next block's operands are loaded into registers while the current one is computed.
struct FwArgs {
  Tensor q, k, v;
  Gate g;
  States s0, sT;
  char* y;                  // [B,T,H,M], contiguous
  const i64* lengths;
  const float* local;       // states that the segments in front leave behind, each from zero; null: one segment
  const double* totals;     // their sums of g
  i64 B, T, H, Hk, M, N, nseg, blocks_per_seg;
  double scale;
};

constexpr int SQ = stride_along(WA), SK = stride_down(WA), SV = stride_down(64), SP = stride_along(L);
constexpr int LT = L / 16, NT = WA / 16;

extern "C" __global__ void __launch_bounds__(256, 2) la_fw(FwArgs a) {
  __shared__ __attribute__((aligned(16))) u16 Q[RP * L * SQ], K[RP * L * SK], V[RP * L * SV], P[RP * L * SP];
  __shared__ Decays<L> D;
  const int tid = threadIdx.x, lane = tid & 63, p = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nmt = (int)((a.M + 63) / 64);
  i64 group;
  int mt;
  if (!spread(blockIdx.x, nmt, a.B * a.H * a.nseg, &group, &mt)) return;
  const i64 bh = group / a.nseg, seg = group % a.nseg, b = bh / a.H, h = bh % a.H, hk = h / (a.H / a.Hk);
  const int m0 = mt * 64, mw = m0 + 16 * w;
  const i64 len = length_of(a.lengths, b, a.T);
  const i64 first = seg * a.blocks_per_seg, nblocks = (a.T + L - 1) / L;
  const i64 last = first + a.blocks_per_seg < nblocks ? first + a.blocks_per_seg : nblocks;

  f4 S[NT];                 // S^T: column m = mw + p, rows n = 16 nt + 4 g + r
  for (int nt = 0; nt < NT; nt++)
    for (int r = 0; r < 4; r++) {
      const int n = 16 * nt + 4 * g + r, m = mw + p;
      S[nt][r] = a.s0.p && m < a.M && n < a.N ? load_type(a.s0.p, b * a.s0.sb + h * a.s0.sh + m * a.s0.sm + n * a.s0.sn, (int)a.s0.type) : 0.f;
    }
  for (i64 s = 0; s < seg; s++) {                // the state at this segment's start
    const i64 at = bh * (a.nseg - 1) + s;
    const float e = expf((float)a.totals[at]);
    const f4* from = (const f4*)a.local + (at * nmt * 4 + mt * 4 + w) * (NT * 64) + lane;
    for (int nt = 0; nt < NT; nt++) S[nt] = S[nt] * e + from[nt * 64];
  }
  // (tiles above the diagonal stay zero)
  for (int i = tid; i < RP * L * SP / 8; i += 256) *(v4u*)(P + 8 * i) = v4u{0, 0, 0, 0};

  const char* qb = a.q.p + (b * a.q.sb + hk * a.q.sh) * ESZ;
  const char* kb = a.k.p + (b * a.k.sb + hk * a.k.sh) * ESZ;
  const char* vb = a.v.p + (b * a.v.sb + h * a.v.sh + m0 * a.v.sn) * ESZ;
  const int vcols = a.M - m0 < 64 ? (int)(a.M - m0) : 64;
  Staging<WA, SQ, L, 256> rq;
  Staging<WA, SK, L, 256> rk;
  Staging<64, SV, L, 256> rv;
  double rg = 0.0;
  const auto fetch = [&](i64 c) {
    const i64 t0 = c * L;
    const int rows = len - t0 < L ? (int)(len - t0) : L;       // (may be negative)
    rq.load(qb + t0 * a.q.st * ESZ, a.q, rows, (int)a.N, tid);
    rk.load(kb + t0 * a.k.st * ESZ, a.k, rows, (int)a.N, tid);
    rv.load(vb + t0 * a.v.st * ESZ, a.v, rows, vcols, tid);
    rg = tid < L && tid < rows ? gate_of(a.g, b, h, t0 + tid) : 0.0;
  };
  if (first < last) fetch(first);
  for (i64 c = first; c < last; c++) {
    const i64 t0 = c * L;
    __syncthreads();
    rq.store(Q, tid);
    rk.store(K, tid);
    rv.store(V, tid);
    if (w == 0) fill_decays<L>(D, rg, lane);
    if (c + 1 < last) fetch(c + 1);
    __syncthreads();
    for (int idx = w; idx < LT * (LT + 1) / 2; idx += 4) {
      int it, jt;
      tile_of(idx, &it, &jt);
      f4 x = {0.f, 0.f, 0.f, 0.f};               // column i = 16 it + p, rows j = 16 jt + 4 g + r
#pragma unroll
      for (int ks = 0; ks < WA / 32; ks++)
        x = mul<RAW>(along8<SK, L>(K, 16 * jt + p, 32 * ks, g), along8<SQ, L>(Q, 16 * it + p, 32 * ks, g), x);
      const int i = 16 * it + p;
      const float hi = D.hi[i], lo = D.lo[i];
      for (int r = 0; r < 4; r++) {
        const int j = 16 * jt + 4 * g + r;
        x[r] = j <= i ? x[r] * decay_between(D, hi, lo, j) : 0.f;
      }
      u32 d[RP * 2];
      split2<RP>(x[0], x[1], d, 2);
      split2<RP>(x[2], x[3], d + 1, 2);
      for (int q = 0; q < RP; q++) *(v2u*)(P + (q * L + i) * SP + 16 * jt + 4 * g) = v2u{d[2 * q], d[2 * q + 1]};
    }
    __syncthreads();
    f4 y[LT];                                    // y^T: column i = 16 it + p, rows m = mw + 4 g + r
    for (int it = 0; it < LT; it++) y[it] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < WA / 32; ks++) {
      float x[8];
      for (int r = 0; r < 4; r++) {
        x[r] = S[2 * ks][r];
        x[4 + r] = S[2 * ks + 1][r];
      }
      const Frag<RP> s = make_frag<RP>(x);
#pragma unroll
      for (int it = 0; it < LT; it++) y[it] = mul<CALC>(s, along<SQ, L>(Q, 16 * it + p, 32 * ks, g), y[it]);
    }
    for (int it = 0; it < LT; it++) y[it] *= D.from_start[16 * it + p];
    const float all = D.all;
    for (int nt = 0; nt < NT; nt++) S[nt] *= all;
#pragma unroll
    for (int jb = 0; jb < L / 32; jb++) {
      const Frag<RP> vf = down<SV, L>(V, 32 * jb, 16 * w, lane);
#pragma unroll
      for (int it = 2 * jb; it < LT; it++) y[it] = mul<CALC>(vf, along<SP, L>(P, 16 * it + p, 32 * jb, g), y[it]);
      float x[8];
      frag_values(vf, x);
      const f4 e0 = *(const f4*)(D.to_end + 32 * jb + 4 * g), e1 = *(const f4*)(D.to_end + 32 * jb + 16 + 4 * g);
      for (int r = 0; r < 4; r++) {
        x[r] *= e0[r];
        x[4 + r] *= e1[r];
      }
      const Frag<3> vd = make_frag<3>(x);
#pragma unroll
      for (int nt = 0; nt < NT; nt++) S[nt] = mul<2>(down<SK, L>(K, 32 * jb, 16 * nt, lane), vd, S[nt]);
    }
    const float scale = (float)a.scale;
    for (int it = 0; it < LT; it++) {
      const i64 t = t0 + 16 * it + p;
      const int m = mw + 4 * g;
      if (t >= a.T || m >= a.M) continue;
      f4 o = y[it] * scale;
      if (t >= len) o = f4{0.f, 0.f, 0.f, 0.f};
      char* at = a.y + (((b * a.T + t) * a.H + h) * a.M + m) * ESZ;
      if (a.M % 4 == 0) {
        if constexpr (IN == FP32) *(f4*)at = o;
        else if constexpr (IN == BF16) *(v2u*)at = v2u{pack_rne(o[0], o[1]), pack_rne(o[2], o[3])};
        else {
          typedef _Float16 h4 __attribute__((ext_vector_type(4)));
          *(h4*)at = __builtin_convertvector(o, h4);
        }
      } else {
        for (int r = 0; r < 4; r++)
          if (m + r < a.M) store_type(at, r, IN, o[r]);
      }
    }
  }
  if (seg == a.nseg - 1)
    for (int nt = 0; nt < NT; nt++)
      for (int r = 0; r < 4; r++) {
        const int n = 16 * nt + 4 * g + r, m = mw + p;
        if (m < a.M && n < a.N) store_type(a.sT.p, b * a.sT.sb + h * a.sT.sh + m * a.sT.sm + n * a.sT.sn, (int)a.sT.type, S[nt][r]);
      }
}
#endif

// ================================================================== states only
#ifdef KERNEL_WALK
// X' = exp(G_L) X + sum_t e_t a_t b_t^T over the blocks of a sequence, forwards (e_t = exp(G_L - G_t): the state itself)
// or backwards (e_t = scale exp(G_t): the state's gradient, from a = dy, b = q).  One workgroup holds 64 of b's columns,
// wave w 16 of them times all WA of a's.  Two uses: what a segment leaves behind (`local`, from zero), and the
// value in front of every block (`marks`) for the gradient kernel; both as accumulator tiles, fp32, in lane order.
struct Job {
  Tensor a, b;              // [B,T,heads,width]
  States init, fin;         // sm: stride of a's index, sn: of b's
  float* marks;
  float* local;
  double* totals;
  i64 Wa, Wb, Ha, Hb;       // widths and heads of a and b
  i64 back;
};
struct WalkArgs {
  Job job[2];
  Gate g;
  const i64* lengths;
  i64 B, T, H, nseg, blocks_per_seg, only_local, cols_tiles;
  double scale;
};

constexpr int SA = stride_down(WA), SB = stride_down(64);
constexpr int AT = WA / 16;

extern "C" __global__ void __launch_bounds__(256, 2) la_walk(WalkArgs args) {
  __shared__ __attribute__((aligned(16))) u16 A[RP * L * SA], Bt[RP * L * SB];
  __shared__ Decays<L> D;
  const Job& j = args.job[blockIdx.y];
  const int tid = threadIdx.x, lane = tid & 63, p = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const i64 nseg = args.only_local ? args.nseg - 1 : args.nseg;
  const int nct = (int)((j.Wb + 63) / 64);
  i64 group;
  int ct;
  if (!spread(blockIdx.x, (int)args.cols_tiles, args.B * args.H * nseg, &group, &ct) || ct >= nct) return;
  const i64 bh = group / nseg, seg = group % nseg, b = bh / args.H, h = bh % args.H;
  const i64 len = length_of(args.lengths, b, args.T);
  const i64 nblocks = (args.T + L - 1) / L;
  const i64 first = seg * args.blocks_per_seg;
  const i64 last = first + args.blocks_per_seg < nblocks ? first + args.blocks_per_seg : nblocks;
  const int c0 = ct * 64, cw = c0 + 16 * w;

  f4 X[AT];                 // column cw + p of b, rows 16 at + 4 g + r of a
  for (int at = 0; at < AT; at++)
    for (int r = 0; r < 4; r++) {
      const int row = 16 * at + 4 * g + r, col = cw + p;
      X[at][r] = !args.only_local && j.init.p && row < j.Wa && col < j.Wb
                     ? load_type(j.init.p, b * j.init.sb + h * j.init.sh + row * j.init.sm + col * j.init.sn, (int)j.init.type) : 0.f;
    }
  if (!args.only_local)
    for (i64 s = 0; s < seg; s++) {
      const i64 at0 = bh * (args.nseg - 1) + s;
      const float e = expf((float)j.totals[at0]);
      const f4* from = (const f4*)j.local + (at0 * nct * 4 + ct * 4 + w) * (AT * 64) + lane;
      for (int at = 0; at < AT; at++) X[at] = X[at] * e + from[at * 64];
    }

  const char* ab = j.a.p + (b * j.a.sb + h / (args.H / j.Ha) * j.a.sh) * ESZ;
  const char* bb = j.b.p + (b * j.b.sb + h / (args.H / j.Hb) * j.b.sh + c0 * j.b.sn) * ESZ;
  const int bcols = j.Wb - c0 < 64 ? (int)(j.Wb - c0) : 64;
  Staging<WA, SA, L, 256> ra;
  Staging<64, SB, L, 256> rb;
  double rg = 0.0, total = 0.0;
  const auto fetch = [&](i64 o) {
    const i64 t0 = (j.back ? nblocks - 1 - o : o) * L;
    const int rows = len - t0 < L ? (int)(len - t0) : L;
    ra.load(ab + t0 * j.a.st * ESZ, j.a, rows, (int)j.Wa, tid);
    rb.load(bb + t0 * j.b.st * ESZ, j.b, rows, bcols, tid);
    rg = tid < L && tid < rows ? gate_of(args.g, b, h, t0 + tid) : 0.0;
  };
  const float scale = j.back ? (float)args.scale : 1.f;
  if (first < last) fetch(first);
  for (i64 o = first; o < last; o++) {
    __syncthreads();
    ra.store(A, tid);
    rb.store(Bt, tid);
    if (w == 0) total += fill_decays<L>(D, rg, lane);
    if (o + 1 < last) fetch(o + 1);
    if (!args.only_local && j.marks && cw < j.Wb) {
      const i64 c = j.back ? nblocks - 1 - o : o;
      f4* to = (f4*)j.marks + ((bh * nblocks + c) * ((j.Wb + 15) / 16) + cw / 16) * (AT * 64) + lane;
      for (int at = 0; at < AT; at++) to[at * 64] = X[at];
    }
    __syncthreads();
    const float all = D.all;
    for (int at = 0; at < AT; at++) X[at] *= all;
#pragma unroll
    for (int jb = 0; jb < L / 32; jb++) {
      float x[8];
      frag_values(down<SB, L>(Bt, 32 * jb, 16 * w, lane), x);
      const float* e = j.back ? D.from_start : D.to_end;
      for (int r = 0; r < 4; r++) {
        x[r] *= scale * e[32 * jb + 4 * g + r];
        x[4 + r] *= scale * e[32 * jb + 16 + 4 * g + r];
      }
      const Frag<3> bd = make_frag<3>(x);
#pragma unroll
      for (int at = 0; at < AT; at++) X[at] = mul<2>(down<SA, L>(A, 32 * jb, 16 * at, lane), bd, X[at]);
    }
  }
  if (args.only_local) {
    const i64 at0 = bh * (args.nseg - 1) + seg;
    f4* to = (f4*)j.local + (at0 * nct * 4 + ct * 4 + w) * (AT * 64) + lane;
    for (int at = 0; at < AT; at++) to[at * 64] = X[at];
    if (tid == 0 && ct == 0) j.totals[at0] = total;
  } else if (j.fin.p && seg == args.nseg - 1) {
    for (int at = 0; at < AT; at++)
      for (int r = 0; r < 4; r++) {
        const int row = 16 * at + 4 * g + r, col = cw + p;
        if (row < j.Wa && col < j.Wb) store_type(j.fin.p, b * j.fin.sb + h * j.fin.sh + row * j.fin.sm + col * j.fin.sn, (int)j.fin.type, X[at][r]);
      }
  }
}
#endif

// ================================================================== gradients
#ifdef KERNEL_GRAD
// One workgroup per (batch, shared head, slice of the heads that share it, block).  With E = exp(G_i - G_j) for i >= j,
// P = (q_i.k_j) E, R = (dy_i.v_j) E scale, and the marks S (state in front) and X (gradient of the state behind):
//   dq_i = sum_j R_ij k_j + scale exp(G_i) S^T dy_i        dk_j = sum_i R_ij q_i + exp(G_L - G_j) X^T v_j
//   dv_j = scale sum_i P_ij dy_i + exp(G_L - G_j) X k_j
//   dg_t = sum_{i>=t>j} P_ij (dy_i.v_j) scale + sum_{i>=t} q_i.dq^S_i + sum_{j<t} k_j.dk^X_j + exp(G_L) <X, S>
// (the last line: the gradient of a step's logarithm is what the step carries over; no term is the difference of two sums
// over the whole sequence, so slow and fast decays alike keep their precision).  Wave w owns every NW-th tile of 16 result
// columns; marks come straight from memory in operand order.  Two operand tiles are in LDS at a time (q, k; then v, dy;
// then k, q), which leaves room for two workgroups per compute unit to cover each other's loads.
struct GradArgs {
  Tensor q, k, v, dy;
  Gate g;
  const float* marks_s;     // [B*H][blocks][ceil(N/16)][WA/16][64][4]
  const float* marks_x;
  char *dq, *dk;            // [slices][B,T,Hk,N]: of the inputs' type with one slice, fp32 with more
  char* dv;                 // [B,T,H,M]
  char* dg;                 // [B,T,H] of type dg_type, or null
  const i64* lengths;
  i64 B, T, H, Hk, M, N, slices, dg_type;
  double scale;
};

// WA: padded M, WB: padded N
constexpr int TH = NW * 64;
constexpr int WX = WA > WB ? WA : WB;
constexpr int SX = stride_down(WX), SP = stride_along(L);
constexpr int LT = L / 16, MT = WA / 16, NT = WB / 16;
constexpr int NTW = (NT + NW - 1) / NW, MTW = (MT + NW - 1) / NW;
constexpr int TILES = LT * (LT + 1) / 2, TPW = (TILES + NW - 1) / NW;

DEV void store4(char* at, int type, f4 o, int n, int N) {
  if (N % 4 == 0) {
    if (type == FP32) *(f4*)at = o;
    else if (type == BF16) *(v2u*)at = v2u{pack_rne(o[0], o[1]), pack_rne(o[2], o[3])};
    else {
      typedef _Float16 h4 __attribute__((ext_vector_type(4)));
      *(h4*)at = __builtin_convertvector(o, h4);
    }
  } else {
    for (int r = 0; r < 4; r++)
      if (n + r < N) store_type(at, r, type, o[r]);
  }
}

extern "C" __global__ void __launch_bounds__(TH, 2) la_grad(GradArgs a) {
  __shared__ __attribute__((aligned(16))) u16 X0[RP * L * SX], X1[RP * L * SX], P[RP * L * SP], R[RP * L * SP];
  __shared__ Decays<L> D;
  __shared__ float rows_pw[LT][L], cols_pw[LT][L], aq[NW][L], bk[NW][L], cs[NW];
  const int tid = threadIdx.x, lane = tid & 63, p = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const i64 nblocks = (a.T + L - 1) / L;
  const i64 share = a.H / a.Hk, per = (share + a.slices - 1) / a.slices;
  const i64 id = blockIdx.x;
  const i64 c = id % nblocks, sl = id / nblocks % a.slices, bhk = id / nblocks / a.slices, b = bhk / a.Hk, hk = bhk % a.Hk;
  const i64 len = length_of(a.lengths, b, a.T), t0 = c * L;
  const int rows = len - t0 < L ? (int)(len - t0) : L, rows_out = a.T - t0 < L ? (int)(a.T - t0) : L;
  const float scale = (float)a.scale;
  const int M = (int)a.M, N = (int)a.N;

  for (int i = tid; i < RP * L * SP / 8; i += TH) {
    *(v4u*)(P + 8 * i) = v4u{0, 0, 0, 0};
    *(v4u*)(R + 8 * i) = v4u{0, 0, 0, 0};
  }
  for (int i = tid; i < LT * L; i += TH) (&rows_pw[0][0])[i] = (&cols_pw[0][0])[i] = 0.f;

  const char* qb = a.q.p + (b * a.q.sb + hk * a.q.sh + t0 * a.q.st) * ESZ;
  const char* kb = a.k.p + (b * a.k.sb + hk * a.k.sh + t0 * a.k.st) * ESZ;
  f4 dq[NTW][LT], dk[NTW][LT];                   // column i (j) = 16 t + p, rows n = 16 nt + 4 g + r
  for (int x = 0; x < NTW; x++)
    for (int t = 0; t < LT; t++) dq[x][t] = dk[x][t] = f4{0.f, 0.f, 0.f, 0.f};

  const i64 h1 = (sl + 1) * per < share ? (sl + 1) * per : share;
  for (i64 hh = sl * per; hh < h1; hh++) {
    const i64 h = hk * share + hh, bh = b * a.H + h;
    const char* vb = a.v.p + (b * a.v.sb + h * a.v.sh + t0 * a.v.st) * ESZ;
    const char* yb = a.dy.p + (b * a.dy.sb + h * a.dy.sh + t0 * a.dy.st) * ESZ;
    const f4* ms = (const f4*)a.marks_s + (bh * nblocks + c) * ((N + 15) / 16) * (MT * 64);
    const f4* mx = (const f4*)a.marks_x + (bh * nblocks + c) * ((N + 15) / 16) * (MT * 64);
    {
      Staging<WB, SX, L, TH> rq, rk;
      rq.load(qb, a.q, rows, N, tid);
      rk.load(kb, a.k, rows, N, tid);
      const double rg = tid < L && tid < rows ? gate_of(a.g, b, h, t0 + tid) : 0.0;
      __syncthreads();
      rq.store(X0, tid);
      rk.store(X1, tid);
      if (w == 0) fill_decays<L>(D, rg, lane);
    }
    Staging<WA, SX, L, TH> rv, ry;
    rv.load(vb, a.v, rows, M, tid);
    ry.load(yb, a.dy, rows, M, tid);
    __syncthreads();
    f4 A[TPW];                                   // q_i.k_j: column i = 16 it + p, rows j = 16 jt + 4 g + r
#pragma unroll
    for (int x = 0; x < TPW; x++) {
      const int idx = w + x * NW;
      A[x] = f4{0.f, 0.f, 0.f, 0.f};
      if (idx < TILES) {
        int it, jt;
        tile_of(idx, &it, &jt);
#pragma unroll
        for (int ks = 0; ks < WB / 32; ks++)
          A[x] = mul<RAW>(along8<SX, L>(X1, 16 * jt + p, 32 * ks, g), along8<SX, L>(X0, 16 * it + p, 32 * ks, g), A[x]);
      }
    }
    __syncthreads();
    rv.store(X0, tid);
    ry.store(X1, tid);
    __syncthreads();
#pragma unroll
    for (int x = 0; x < TPW; x++) {
      const int idx = w + x * NW;
      if (idx >= TILES) continue;
      int it, jt;
      tile_of(idx, &it, &jt);
      f4 W = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < WA / 32; ks++)
        W = mul<RAW>(along8<SX, L>(X0, 16 * jt + p, 32 * ks, g), along8<SX, L>(X1, 16 * it + p, 32 * ks, g), W);
      const int i = 16 * it + p;
      const float hi = D.hi[i], lo = D.lo[i];
      float of_row = 0.f;
      f4 pw, pe, re;
      for (int r = 0; r < 4; r++) {
        const int j = 16 * jt + 4 * g + r;
        const float e = j <= i ? decay_between(D, hi, lo, j) * scale : 0.f;
        pe[r] = j <= i ? A[x][r] * e : 0.f;
        re[r] = j <= i ? W[r] * e : 0.f;
        pw[r] = j <= i ? pe[r] * W[r] : 0.f;
        of_row += pw[r];
      }
      u32 d[RP * 2], f[RP * 2];
      split2<RP>(pe[0], pe[1], d, 2);
      split2<RP>(pe[2], pe[3], d + 1, 2);
      split2<RP>(re[0], re[1], f, 2);
      split2<RP>(re[2], re[3], f + 1, 2);
      for (int q = 0; q < RP; q++) {
        *(v2u*)(P + (q * L + i) * SP + 16 * jt + 4 * g) = v2u{d[2 * q], d[2 * q + 1]};
        *(v2u*)(R + (q * L + i) * SP + 16 * jt + 4 * g) = v2u{f[2 * q], f[2 * q + 1]};
      }
      if (a.dg) {
        of_row = sum_groups(of_row);
        if (g == 0) rows_pw[jt][i] = of_row;
        for (int r = 0; r < 4; r++) {
          const float s = sum16(pw[r]);
          if (p == 0) cols_pw[it][16 * jt + 4 * g + r] = s;
        }
      }
    }
    __syncthreads();
    // with v in X0, dy in X1: what the marks give to dq and dk, and the block's own share of dv
    f4 qs[NTW][LT], kx[NTW][LT], dv[MTW][LT];
    float inner = 0.f;
#pragma unroll
    for (int x = 0; x < NTW; x++) {
      const int nt = w + x * NW;
      for (int t = 0; t < LT; t++) qs[x][t] = kx[x][t] = f4{0.f, 0.f, 0.f, 0.f};
      if (16 * nt >= N) continue;
#pragma unroll
      for (int ks = 0; ks < WA / 32; ks++) {
        const f4 s0 = ms[(nt * MT + 2 * ks) * 64 + lane], s1 = ms[(nt * MT + 2 * ks + 1) * 64 + lane];
        const f4 x0 = mx[(nt * MT + 2 * ks) * 64 + lane], x1 = mx[(nt * MT + 2 * ks + 1) * 64 + lane];
        float s[8], y[8];
        for (int r = 0; r < 4; r++) {
          s[r] = s0[r];
          s[4 + r] = s1[r];
          y[r] = x0[r];
          y[4 + r] = x1[r];
          inner += s0[r] * x0[r] + s1[r] * x1[r];
        }
        const Frag<3> sf = make_frag<3>(s), xf = make_frag<3>(y);
#pragma unroll
        for (int t = 0; t < LT; t++) {
          qs[x][t] = mul<2>(sf, along<SX, L>(X1, 16 * t + p, 32 * ks, g), qs[x][t]);
          kx[x][t] = mul<2>(xf, along<SX, L>(X0, 16 * t + p, 32 * ks, g), kx[x][t]);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < MTW; x++) {
      const int mt = w + x * NW;
      for (int t = 0; t < LT; t++) dv[x][t] = f4{0.f, 0.f, 0.f, 0.f};
      if (16 * mt >= M) continue;
#pragma unroll
      for (int ib = 0; ib < L / 32; ib++) {
        const Frag<RP> yf = down<SX, L>(X1, 32 * ib, 16 * mt, lane);
#pragma unroll
        for (int t = 0; t < LT; t++)
          if (16 * t < 32 * ib + 32) dv[x][t] = mul<CALC>(yf, down<SP, L>(P, 32 * ib, 16 * t, lane), dv[x][t]);
      }
    }
    {
      Staging<WB, SX, L, TH> rq, rk;
      rq.load(qb, a.q, rows, N, tid);
      rk.load(kb, a.k, rows, N, tid);
      __syncthreads();
      rk.store(X0, tid);
      rq.store(X1, tid);
    }
    __syncthreads();
    // with k in X0, q in X1
#pragma unroll
    for (int t = 0; t < LT; t++) {
      const float from = D.from_start[16 * t + p] * scale, to = D.to_end[16 * t + p];
      float sq = 0.f, sk = 0.f;
#pragma unroll
      for (int x = 0; x < NTW; x++) {
        const int nt = w + x * NW;
        if (nt >= NT) continue;
        qs[x][t] *= from;
        kx[x][t] *= to;
        if (a.dg) {
          for (int q = 0; q < RP; q++) {
            const v2u qv = *(const v2u*)(X1 + (q * L + 16 * t + p) * SX + 16 * nt + 4 * g);
            const v2u kv = *(const v2u*)(X0 + (q * L + 16 * t + p) * SX + 16 * nt + 4 * g);
            sq += qs[x][t][0] * as_f(qv[0] << 16) + qs[x][t][1] * as_f(qv[0] & 0xffff0000u) + qs[x][t][2] * as_f(qv[1] << 16) + qs[x][t][3] * as_f(qv[1] & 0xffff0000u);
            sk += kx[x][t][0] * as_f(kv[0] << 16) + kx[x][t][1] * as_f(kv[0] & 0xffff0000u) + kx[x][t][2] * as_f(kv[1] << 16) + kx[x][t][3] * as_f(kv[1] & 0xffff0000u);
          }
        }
        dq[x][t] += qs[x][t];
        dk[x][t] += kx[x][t];
      }
      if (a.dg) {
        sq = sum_groups(sq);
        sk = sum_groups(sk);
        if (g == 0) {
          aq[w][16 * t + p] = sq;
          bk[w][16 * t + p] = sk;
        }
      }
    }
    if (a.dg) {
      inner = sum_groups(sum16(inner));
      if (lane == 0) cs[w] = inner;
    }
#pragma unroll
    for (int x = 0; x < NTW; x++) {
      const int nt = w + x * NW;
      if (16 * nt >= N) continue;
#pragma unroll
      for (int tb = 0; tb < L / 32; tb++) {
        const Frag<RP> kf = down<SX, L>(X0, 32 * tb, 16 * nt, lane), qf = down<SX, L>(X1, 32 * tb, 16 * nt, lane);
#pragma unroll
        for (int t = 0; t < LT; t++) {
          if (t >= 2 * tb) dq[x][t] = mul<CALC>(kf, along<SP, L>(R, 16 * t + p, 32 * tb, g), dq[x][t]);
          if (16 * t < 32 * tb + 32) dk[x][t] = mul<CALC>(qf, down<SP, L>(R, 32 * tb, 16 * t, lane), dk[x][t]);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < MTW; x++) {
      const int mt = w + x * NW;
      if (16 * mt >= M) continue;
      f4 e[LT];
      for (int t = 0; t < LT; t++) e[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < WB / 32; ks++) {
        // lane p holds row m = 16 mt + p, columns n = 32 ks + {4g.., 16 + 4g..}: the marks' tiles read across
        float s[8];
        for (int r = 0; r < 8; r++) {
          const int nt = 2 * ks + r / 4;
          const float* at = (const float*)(mx + (nt * MT + mt) * 64 + (p >> 2) * 16 + 4 * g + r % 4) + (p & 3);
          s[r] = 16 * nt < N ? *at : 0.f;
        }
        const Frag<RP> xf = make_frag<RP>(s);
#pragma unroll
        for (int t = 0; t < LT; t++) e[t] = mul<CALC>(xf, along<SX, L>(X0, 16 * t + p, 32 * ks, g), e[t]);
      }
      for (int t = 0; t < LT; t++) {
        const int j = 16 * t + p, m = 16 * mt + 4 * g;
        if (j >= rows_out || m >= M) continue;
        f4 o = dv[x][t] + e[t] * D.to_end[j];
        if (j >= rows) o = f4{0.f, 0.f, 0.f, 0.f};
        store4(a.dv + (((b * a.T + t0 + j) * a.H + h) * M + m) * ESZ, IN, o, m, M);
      }
    }
    if (a.dg) {
      __syncthreads();
      if (w == 0) {
        double x = 0.0, y = 0.0, z = 0.0;
        if (lane < L) {
          for (int t = 0; t < LT; t++) x += (double)rows_pw[t][lane] - (double)cols_pw[t][lane];
          for (int q = 0; q < NW; q++) {
            x += aq[q][lane];
            y += bk[q][lane];
          }
        }
        for (int q = 0; q < NW; q++) z += cs[q];
        // sum over i >= t of x_i, over j < t of y_j
        const double sx = scan64(x), sy = scan64(y);
        const double dg = (last_lane(sx) - sx + x) + (sy - y) + (double)D.all * z;
        if (lane < rows_out)
          store_type(a.dg, (b * a.T + t0 + lane) * a.H + h, (int)a.dg_type, lane < rows ? (float)dg : 0.f);
      }
    }
  }
  const int type = a.slices == 1 ? IN : FP32;
  const i64 size = type == FP32 ? 4 : 2, skip = a.slices == 1 ? 0 : sl * a.B * a.T * a.Hk * a.N;
#pragma unroll
  for (int x = 0; x < NTW; x++) {
    const int nt = w + x * NW;
    for (int t = 0; t < LT; t++) {
      const int i = 16 * t + p, n = 16 * nt + 4 * g;
      if (i >= rows_out || n >= N) continue;
      const i64 at = (skip + ((b * a.T + t0 + i) * a.Hk + hk) * N + n) * size;
      const bool in = i < rows;
      const f4 zero = {0.f, 0.f, 0.f, 0.f};
      store4(a.dq + at, type, in ? dq[x][t] : zero, n, N);
      store4(a.dk + at, type, in ? dk[x][t] : zero, n, N);
    }
  }
}
#endif

// ================================================================== one token
#ifdef KERNEL_STEP
// S = exp(g) S + v k^T in place, y = scale S q.  Bound by reading and writing the state once.  A group of GL lanes owns a
// row of the state, each lane VE neighbouring columns of it per turn (16 bytes where layout and type allow).
struct StepArgs {
  Tensor q, k, v;           // st unused
  Gate g;
  States s;
  char* y;                  // [B,H,M]
  i64 B, H, Hk, M, N, vec, gl, rows;      // rows of the state per workgroup
  double scale;
};
DEV float load_in(const char* p, i64 i) { return load_type(p, i, IN); }

template <int TYPE, int VE>
DEV void step_rows(const StepArgs& a, i64 b, i64 h, int r0, int tid) {
  const int gl = (int)a.gl, sub = tid % gl, grp = tid / gl, groups = 256 / gl;
  const i64 hk = h / (a.H / a.Hk);
  const float e = expf((float)gate_of(a.g, b, h, 0)), scale = (float)a.scale;
  const char* qp = a.q.p + (b * a.q.sb + hk * a.q.sh) * ESZ;
  const char* kp = a.k.p + (b * a.k.sb + hk * a.k.sh) * ESZ;
  const char* vp = a.v.p + (b * a.v.sb + h * a.v.sh) * ESZ;
  constexpr int SZ = TYPE == FP32 ? 4 : 2;
  const int M = (int)a.M, N = (int)a.N;
  const int end = r0 + (int)a.rows < M ? r0 + (int)a.rows : M;
  for (int m = r0 + grp; m < ((end - r0 + groups - 1) / groups) * groups + r0; m += groups) {
    float acc = 0.f;
    if (m < end) {
      const float v = load_in(vp, m * a.v.sn);
      char* row = a.s.p + (b * a.s.sb + h * a.s.sh + m * a.s.sm) * SZ;
      for (int n = sub * VE; n < N; n += gl * VE) {
        float s[VE];
        if constexpr (VE == 1) {
          s[0] = load_type(row, n * a.s.sn, TYPE);
        } else if constexpr (TYPE == FP32) {
          const f4 t = *(const f4*)(row + n * 4);
          for (int i = 0; i < 4; i++) s[i] = t[i];
        } else {
          const v4u t = *(const v4u*)(row + n * 2);
          for (int i = 0; i < VE; i++) {
            const u16 x = (u16)(t[i / 2] >> (i % 2 * 16));
            s[i] = TYPE == FP16 ? half_to_f(x) : as_f((u32)x << 16);
          }
        }
        for (int i = 0; i < VE; i++) {
          s[i] = e * s[i] + v * load_in(kp, (n + i) * a.k.sn);
          acc += s[i] * load_in(qp, (n + i) * a.q.sn);
        }
        if constexpr (VE == 1) {
          store_type(row, n * a.s.sn, TYPE, s[0]);
        } else if constexpr (TYPE == FP32) {
          *(f4*)(row + n * 4) = f4{s[0], s[1], s[2], s[3]};
        } else {
          v4u t;
          for (int i = 0; i < VE / 2; i++) {
            if constexpr (TYPE == BF16) t[i] = pack_rne(s[2 * i], s[2 * i + 1]);
            else t[i] = (u32)__builtin_bit_cast(u16, (_Float16)s[2 * i]) | (u32)__builtin_bit_cast(u16, (_Float16)s[2 * i + 1]) << 16;
          }
          *(v4u*)(row + n * 2) = t;
        }
      }
    }
    for (int x = 1; x < gl; x <<= 1) acc += __shfl_xor(acc, x, 64);
    if (m < end && sub == 0) store_type(a.y, (b * a.H + h) * M + m, IN, acc * scale);
  }
}

extern "C" __global__ void __launch_bounds__(256) la_step(StepArgs a) {
  const i64 per = (a.M + a.rows - 1) / a.rows;
  const i64 bh = blockIdx.x / per;
  const int r0 = (int)(blockIdx.x % per * a.rows);
  const i64 b = bh / a.H, h = bh % a.H;
  const int tid = threadIdx.x;
  if (a.s.type == FP32) {
    if (a.vec) step_rows<FP32, 4>(a, b, h, r0, tid);
    else step_rows<FP32, 1>(a, b, h, r0, tid);
  } else if (a.s.type == BF16) {
    if (a.vec) step_rows<BF16, 8>(a, b, h, r0, tid);
    else step_rows<BF16, 1>(a, b, h, r0, tid);
  } else {
    if (a.vec) step_rows<FP16, 8>(a, b, h, r0, tid);
    else step_rows<FP16, 1>(a, b, h, r0, tid);
  }
}
#endif
