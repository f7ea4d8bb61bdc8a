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
// The gradients are the same walk in other roles (dy already scaled; X the gradient of the state):
//
//     dq_i = sum_{j<=i} exp(G_i - G_j) (dy_i.v_j) k_j + exp(G_i) S^T dy_i              forwards,  (q, k, v) <- (dy, v, k)
//     dk_j = sum_{i>=j} exp(G_i - G_j) (v_j.dy_i) q_i + exp(G_L - G_j) X^T v_j         backwards, (q, k, v) <- (v, dy, q)
//     dv_j = sum_{i>=j} exp(G_i - G_j) (k_j.q_i) dy_i + exp(G_L - G_j) X k_j           backwards, (q, k, v) <- (k, q, dy)
//
// so one kernel, la_block, computes y and all three; backwards, a sequence is read from its end and the decay of a position
// is the one of the token behind it.
//
// Compiled per set of constants by flex_rnn_amd/handwritten.py, which passes
//   KERNEL_BLOCK / KERNEL_GATE / KERNEL_STEP   which kernel this code object holds
//   IN     element type of q, k, v, dy: 0 bfloat16, 1 float16, 2 float32
//   W      padded width (64, 128 or 256) of q and k
//   OUT    0: the state alone (what a segment of a sequence leaves behind)
//   DOTS   1: also what the gradient of g is made of
//   FAST   1: every operand allows 16-byte loads and rows of y are a multiple of four long.  Without the branches and the
//          second set of loads and stores that any other layout needs, a block takes a tenth less time
//   WIDE   with FAST, the type of y: 0 the operands', 1 float32
//   NBUF   operand tiles in LDS: 2 lets a block's operands arrive while the one before is read, 1 saves LDS
//   OCC    waves per SIMD to compile for
//
// Numbers on the matrix cores.  All products are v_mfma_f32_16x16x32_bf16: fp32 sums of bfloat16 factors.  A factor with
// more bits is a sum of RP bfloat16 parts (float16: 2, float32: 3; the parts hold every bit, because each takes the leading
// 8 bits of what is left), and a product of two such factors is the sum of the products of their parts, less those below the
// last bit that counts.  The bfloat16 exponent is that of float32, so nothing overflows on the way that would not in float32.
//   - factors read from memory are exact;
//   - the decayed products P = exp(G_i - G_j) q_i.k_j are rounded to RP parts, and to two with bfloat16: each stands for a whole
//     row of v, so its rounding would not average out (the second part is 2.5 % of a block's time, and y as far from the exact
//     result as its own rounding, 1.7e-3 of its norm, where a fast decay leaves little of the state);
//   - the state, where it is a factor, is rounded to as many parts as P: with one part in bfloat16 an element of y whose terms
//     cancel was off by up to ten times its own rounding (2.2e-3 of y's norm for a long document, against 1.7e-3, for 2.5 to 6.5 %
//     of the time); to three where the product is part of g's gradient, whose type may be float32 with 16-bit inputs;
//   - the decayed v that enters the state has three parts: the state is an fp32 result even where the inputs are not.
// The state itself stays in fp32 accumulators for the whole sequence.
//
// Layout.  Operand tiles sit in LDS as [token][column], one plane per part.  The matrix instruction's reduction index may be
// permuted as long as both factors use the same order; everything here uses the order of its own results - in a block of 32,
// lane group g = lane/16 holds {4g..4g+3, 16+4g..16+4g+3} - so an accumulator tile becomes an operand without leaving
// its registers, and ds_read_b64_tr_b16 delivers the same order for
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

#ifndef FAST
#define FAST 0
#define WIDE 0
#endif

constexpr int ESZ = IN == 2 ? 4 : 2;          // bytes per element of q, k, v, dy
constexpr int RP = IN + 1;                    // bfloat16 parts of such an element
constexpr int L = 32;                         // tokens per block
constexpr double LOG2E = 1.4426950408889634;
constexpr double NO_DECAY = -200.0;           // keeps the sums of logarithms finite
constexpr double ZERO_DECAY = -104.0;         // exp of it and less is zero in fp32

enum { BF16 = 0, FP16 = 1, FP32 = 2 };

struct Tensor {      // strides in elements
  const char* p;
  i64 sb, st, sh, sn;
  i64 vec;           // how 8 neighbours are read: 1 in aligned pieces of 16 bytes; 2 in pieces at any address (at least 8 columns next to each other); 0 one by one
};

struct States {      // element (row, column) of a head's state, of a type; or p = null
  char* p;
  i64 sb, sh, sr, sc, type;
};

DEV float as_f(u32 x) { return __uint_as_float(x); }
DEV u32 as_u(float x) { return __float_as_uint(x); }
DEV float half_to_f(u16 h) { return (float)__builtin_bit_cast(_Float16, h); }

DEV u32 pack_rne(float a, float b) {           // two floats to bfloat16, to nearest even
  f2 v = {a, b};
  return __builtin_bit_cast(u32, __builtin_convertvector(v, bh2));
}
DEV u32 pack_top(float a, float b) { return __builtin_amdgcn_perm(as_u(b), as_u(a), 0x07060302u); }

// NP parts of the two floats a, b: the first by truncation (which never overflows), the last to nearest; what is left is exact.
// With factors of two and three parts, products leave out those of low parts: there the second part is to nearest, too.
// Truncated, it has the number's sign, and so has what is left out: every product of float32 was 4e-8 too small.  (bfloat16
// leaves nothing out, and truncation frees its registers earlier.)
// With INF an infinity is a part by itself; without, it leaves a NaN behind (as its products with zeros would).
template <int NP, bool INF = false>
DEV void split2(float a, float b, u32* out, int stride) {
  for (int i = 0; i < NP - 1; i++) {
    const bool cut = i == 0 || RP == 1;
    const u32 d = cut ? pack_top(a, b) : pack_rne(a, b);
    const float ta = as_f(cut ? as_u(a) & 0xffff0000u : d << 16), tb = as_f((cut ? as_u(b) : d) & 0xffff0000u);
    out[i * stride] = d;
    a = INF && a == ta ? 0.f : a - ta;
    b = INF && b == tb ? 0.f : b - tb;
  }
  out[(NP - 1) * stride] = pack_rne(a, b);
}

template <int NP>
struct Frag {        // 8 elements of the reduction index per lane, NP parts
  v4u d[NP];
};

template <int NP, bool INF = false>
DEV Frag<NP> make_frag(const float* x) {
  Frag<NP> f;
  u32 t[NP * 4];
  for (int i = 0; i < 4; i++) split2<NP, INF>(x[2 * i], x[2 * i + 1], t + i, 4);
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
// the same for N left factors, one after the other within a pair of parts: no product waits for the one before it
template <int N, int LIM, int PA, int PB>
DEV void mul_each(const Frag<PA>* a, const Frag<PB>& b, f4* c) {
#pragma unroll
  for (int s = LIM; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < PA; i++) {
      const int j = s - i;
      if (j >= 0 && j < PB)
#pragma unroll
        for (int n = 0; n < N; n++)
          c[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bh8, a[n].d[i]), __builtin_bit_cast(bh8, b.d[j]), c[n], 0, 0, 0);
    }
}
constexpr int RAW = RP == 1 ? 0 : 2;           // both factors exact
constexpr int PP = RP == 1 ? 2 : RP;           // parts of the decayed products, and of the state as a factor

// ------------------------------------------------------------------ LDS tiles
constexpr int stride_down(int w) { return w + 16; }       // for tiles read down their columns
constexpr int stride_along(int w) { return w + 8; }

DEV v4s tr_read(const u16* p) {
  typedef __attribute__((address_space(3))) v4s* lds_ptr;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(__attribute__((address_space(3))) void*)p);
}

// lane (p = lane % 16, g = lane / 16) gets column c0 + p, rows r0 + {4g..4g+3, 16+4g..16+4g+3}
template <int STR>
DEV Frag<RP> down(const u16* tile, int r0, int c0, int lane) {
  const int p = lane & 15, g = lane >> 4;
  const u16* at = tile + (r0 + 4 * g + (p >> 2)) * STR + c0 + 4 * (p & 3);
  Frag<RP> f;
#pragma unroll
  for (int i = 0; i < RP; i++) {
    const v2u a = __builtin_bit_cast(v2u, tr_read(at + i * L * STR));
    const v2u b = __builtin_bit_cast(v2u, tr_read(at + i * L * STR + 16 * STR));
    f.d[i] = v4u{a[0], a[1], b[0], b[1]};
  }
  return f;
}

// lane (p, g) gets row r, columns c0 + {4g..4g+3, 16+4g..16+4g+3}
template <int STR, int NP = RP>
DEV Frag<NP> along(const u16* tile, int r, int c0, int g) {
  const u16* at = tile + r * STR + c0 + 4 * g;
  Frag<NP> f;
#pragma unroll
  for (int i = 0; i < NP; i++) {
    const v2u a = *(const v2u*)(at + i * L * STR), b = *(const v2u*)(at + i * L * STR + 16);
    f.d[i] = v4u{a[0], a[1], b[0], b[1]};
  }
  return f;
}

// lane (p, g) gets row r, columns c0 + 8g..8g+7: where the order is free on both sides
template <int STR>
DEV Frag<RP> along8(const u16* tile, int r, int c0, int g) {
  Frag<RP> f;
#pragma unroll
  for (int i = 0; i < RP; i++) f.d[i] = *(const v4u*)(tile + i * L * STR + r * STR + c0 + 8 * g);
  return f;
}

// ------------------------------------------------------------------ memory to registers
struct Raw {         // 8 elements as they are in memory
  v4u d[ESZ / 2];
};

// A tensor's block of tokens as a buffer: what is not to be read gets an offset behind its end and comes back as zero, so
// nothing outside the tensor is touched and no branch waits.  Offsets are 32 bits within a block; the block's address is 64.
constexpr u32 NOTHING = 0x80000000u;
typedef __amdgpu_buffer_rsrc_t Buffer;
DEV Buffer buffer_at(const char* base) { return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00027000); }

// 8 elements from byte offset `at` on, `step` apart; those from `n` on are zero
DEV Raw load_apart(Buffer base, u32 at, u32 step, int n) {
  Raw r;
  u32 w[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    const u32 off = e < n ? at + e * step : NOTHING;
    if constexpr (ESZ == 4) w[e] = __builtin_amdgcn_raw_buffer_load_b32(base, off, 0, 0);
    else w[e] = (u16)__builtin_amdgcn_raw_buffer_load_b16(base, off, 0, 0);
  }
  if constexpr (ESZ == 4) {
    r.d[0] = v4u{w[0], w[1], w[2], w[3]};
    r.d[ESZ / 2 - 1] = v4u{w[4], w[5], w[6], w[7]};
  } else {
    r.d[0] = v4u{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
  }
  return r;
}

// 8 elements at any address
DEV Raw load_any(const char* at) {
  typedef v4u v4u_any __attribute__((aligned(2)));
  Raw r;
  for (int i = 0; i < ESZ / 2; i++) r.d[i] = ((const v4u_any*)at)[i];
  return r;
}
// the last 8 - n of them first, zeros behind
DEV Raw drop(const Raw& r, int n) {
  Raw o;
  if constexpr (ESZ == 4) {
    u32 x[8];
    for (int e = 0; e < 8; e++) x[e] = r.d[e / 4][e % 4];
    for (int b = 4; b > 0; b /= 2)
      for (int e = 0; e < 8; e++) x[e] = n & b ? (e + b < 8 ? x[e + b < 8 ? e + b : e] : 0u) : x[e];
    for (int e = 0; e < 8; e++) o.d[e / 4][e % 4] = x[e];
  } else {
    u64 lo = (u64)r.d[0][1] << 32 | r.d[0][0], hi = (u64)r.d[0][3] << 32 | r.d[0][2];
    const int bits = 16 * n;
    lo = n >= 4 ? hi >> (bits & 63) : n > 0 ? lo >> bits | hi << (64 - bits) : lo;
    hi = n >= 4 ? 0 : n > 0 ? hi >> bits : hi;
    o.d[0] = v4u{(u32)lo, (u32)(lo >> 32), (u32)hi, (u32)(hi >> 32)};
  }
  return o;
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
    const Frag<RP> f = make_frag<RP, true>(x);
    for (int p = 0; p < RP; p++) *(v4u*)(at + p * PLANE) = f.d[p];
  }
}

// A tile of L tokens x W_ columns, staged by 256 threads, block after block; row r of the tile is token r, or L - 1 - r
// backwards.  A thread's offsets within a block stay the same, only the block's address moves.
template <int W_, int STR>
struct Staging {
  static constexpr int N = L * (W_ / 8) / 256, ROWS = 256 / (W_ / 8);       // pieces of a thread, and the rows between them
  Raw r[N];
  u32 off[N], sn;
  const char* at;           // the next block's first token
  i64 step;
  int token, dir;           // of the thread's first piece
  int vec;
  int left;                 // columns from the thread's own on

  DEV_MEMBER void init(const Tensor& t, const char* first, int cols, bool back, int tid) {
    const int row = tid / (W_ / 8), col = tid % (W_ / 8) * 8;
    const u32 st = (u32)t.st * ESZ;
    sn = (u32)t.sn * ESZ;
    vec = (int)t.vec;
    token = back ? L - 1 - row : row;
    dir = back ? -ROWS : ROWS;
    left = cols - col;
#pragma unroll
    for (int i = 0; i < N; i++) off[i] = left > 0 ? (token + i * dir) * st + col * sn : NOTHING;
    at = first;
    step = (back ? -L : L) * t.st * ESZ;
  }
  // (with vec, columns come in eights: all of a piece's are inside, or none)
  DEV_MEMBER void load(int tokens) {
    const Buffer from = buffer_at(at);
    const char* before = at;
    at += step;
    if (FAST || vec == 1) {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const u32 o = token + i * dir < tokens ? off[i] : NOTHING;
#pragma unroll
        for (int e = 0; e < ESZ / 2; e++) r[i].d[e] = __builtin_amdgcn_raw_buffer_load_b128(from, o + 16 * e, 0, 0);
      }
    } else if (vec == 2) {
      // a row's last piece is read so that it ends with the row, and put right on the way to LDS: nothing waits for it here
#pragma unroll
      for (int i = 0; i < N; i++) {
        for (int e = 0; e < ESZ / 2; e++) r[i].d[e] = v4u{0, 0, 0, 0};
        if (left > 0 && token + i * dir < tokens) r[i] = load_any(before + off[i] - (left < 8 ? (8 - left) * ESZ : 0));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        u32 apart = sn;
        asm volatile("" : "+s"(apart));          // (or eight addresses a piece are kept in registers for this path)
        r[i] = load_apart(from, off[i], apart, token + i * dir < tokens ? left : 0);
      }
    }
  }
  DEV_MEMBER void store(u16* tile, int tid) {
    const int row = tid / (W_ / 8), col = tid % (W_ / 8) * 8;
#pragma unroll
    for (int i = 0; i < N; i++) {
      if (!FAST && vec == 2 && left < 8) r[i] = drop(r[i], left > 0 ? 8 - left : 0);
      store_parts<L * STR>(tile + (row + i * ROWS) * STR + col, r[i]);
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
DEV double scan32(double x) {                  // inclusive sums over either half of the 64 lanes
  x += dpp_or_zero<0x111, 0xf>(x);             // row_shr 1, 2, 4, 8: within rows of 16
  x += dpp_or_zero<0x112, 0xf>(x);
  x += dpp_or_zero<0x114, 0xf>(x);
  x += dpp_or_zero<0x118, 0xf>(x);
  return x + dpp_or_zero<0x142, 0xa>(x);       // an even row's last lane into the odd row behind it
}
DEV double scan64(double x) {                  // over all of them
  x = scan32(x);
  return x + dpp_or_zero<0x143, 0xc>(x);       // lane 31 into the upper half
}
DEV double row_of_16(double x) {               // over 16 lanes, in the last of them
  x += dpp_or_zero<0x111, 0xf>(x);
  x += dpp_or_zero<0x112, 0xf>(x);
  x += dpp_or_zero<0x114, 0xf>(x);
  return x + dpp_or_zero<0x118, 0xf>(x);
}
template <class SWAP>
DEV double add_swapped(double x, SWAP swap) {
  const u64 b = __builtin_bit_cast(u64, x);
  const auto lo = swap((u32)b), hi = swap((u32)(b >> 32));
  return __builtin_bit_cast(double, (u64)(u32)hi[0] << 32 | (u32)lo[0]) + __builtin_bit_cast(double, (u64)(u32)hi[1] << 32 | (u32)lo[1]);
}
DEV double over_rows(double x) {               // over the 4 lanes with the same lane % 16
  x = add_swapped(x, [](u32 u) { return __builtin_amdgcn_permlane16_swap(u, u, false, false); });
  return add_swapped(x, [](u32 u) { return __builtin_amdgcn_permlane32_swap(u, u, false, false); });
}
DEV double read_lane(double x, int lane) {
  const u64 b = __builtin_bit_cast(u64, x);
  const u32 lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __builtin_bit_cast(double, (u64)hi << 32 | lo);
}

struct Gate {        // g: [B,T,H] (or [H]: strides 0)
  const char* p;
  i64 sb, st, sh, type;
};

// as it is in memory: what it means is asked for later, so that nothing waits for it here
DEV u32 raw_gate(const Gate& g, i64 b, i64 h, i64 t) {
  const i64 i = b * g.sb + t * g.st + h * g.sh;
  return g.type == FP32 ? ((const u32*)g.p)[i] : (u32)((const u16*)g.p)[i];
}
DEV double gate_value(const Gate& g, u32 raw) {
  const double x = g.type == FP32 ? as_f(raw) : g.type == FP16 ? half_to_f((u16)raw) : as_f(raw << 16);
  return x < NO_DECAY ? NO_DECAY : x;
}
DEV double gate_of(const Gate& g, i64 b, i64 h, i64 t) { return gate_value(g, raw_gate(g, b, h, t)); }

struct Decays {
  // G * log2(e) as a sum of two floats: differences of far sums keep the precision of near ones
  alignas(16) float hi[L];
  alignas(16) float lo[L];
  alignas(16) float from_start[L];             // exp(G_i); the last one is the whole block's
  alignas(16) float to_end[L];                 // exp(G_L - G_i), times the scale of what enters the state
};

// one wave prepares two blocks: lane i of either half holds token i's g (0 behind the last token); returns the sum of g
DEV double fill_decays(Decays* first, Decays* second, double g, float in_scale, int lane) {
  const double G = scan32(g);
  const double end0 = read_lane(G, 31), end1 = read_lane(G, 63);
  const double G2 = G * LOG2E;
  const float hi = (float)G2;
  Decays* d = lane < L ? first : second;
  const int i = lane & (L - 1);
  d->hi[i] = hi;
  d->lo[i] = (float)(G2 - (double)hi);
  d->from_start[i] = (float)exp(G);
  d->to_end[i] = (float)exp((lane < L ? end0 : end1) - G) * in_scale;
  return end0 + end1;
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

template <int CTRL>
DEV float dpp_add(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// Sums over the 2, 4, 8 and 16 neighbours of a lane (swaps within quads, then mirrors: no LDS), and over the lanes 16 and 32
// further (row swaps), known to all of them.
DEV float sum2(float x) { return dpp_add<0xb1>(x); }
DEV float sum4(float x) { return dpp_add<0x4e>(sum2(x)); }
DEV float sum8(float x) { return dpp_add<0x141>(sum4(x)); }
DEV float sum16(float x) { return dpp_add<0x140>(sum8(x)); }
DEV float sum_rows16(float x) {
  const u32 u = __builtin_bit_cast(u32, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __builtin_bit_cast(float, (u32)r[0]) + __builtin_bit_cast(float, (u32)r[1]);
}
DEV float sum_rows32(float x) {
  const u32 u = __builtin_bit_cast(u32, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (u32)r[0]) + __builtin_bit_cast(float, (u32)r[1]);
}
DEV float sum_groups(float x) { return sum_rows32(sum_rows16(x)); }       // over the 4 lanes with the same lane % 16
DEV float sum_lanes(float x, int lanes) {      // over groups of 1 to 64 lanes, a power of two (the same in a whole wave)
  if (lanes >= 2) x = sum2(x);
  if (lanes >= 4) x = dpp_add<0x4e>(x);
  if (lanes >= 8) x = dpp_add<0x141>(x);
  if (lanes >= 16) x = dpp_add<0x140>(x);
  if (lanes >= 32) x = sum_rows16(x);
  if (lanes >= 64) x = sum_rows32(x);
  return x;
}

// Four neighbours of a block's result, the first n of them inside; in one piece where `whole` says that rows are a multiple
// of four long.  Nothing is written at NOTHING.
DEV void store_wide(Buffer to, u32 off, f4 x, int n, bool whole) {
  if (whole) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, x), to, n > 0 ? off : NOTHING, 0, 0);
  else
    for (int r = 0; r < 4; r++) __builtin_amdgcn_raw_buffer_store_b32(as_u(x[r]), to, r < n ? off + 4 * r : NOTHING, 0, 0);
}
DEV void store_in(Buffer to, u32 off, f4 x, int n, bool whole) {
  if constexpr (IN == FP32) {
    store_wide(to, off, x, n, whole);
  } else {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    v2u d;
    if constexpr (IN == BF16) d = v2u{pack_rne(x[0], x[1]), pack_rne(x[2], x[3])};
    else d = __builtin_bit_cast(v2u, __builtin_convertvector(x, h4));
    if (whole) __builtin_amdgcn_raw_buffer_store_b64(d, to, n > 0 ? off : NOTHING, 0, 0);
    else
      for (int r = 0; r < 4; r++) __builtin_amdgcn_raw_buffer_store_b16((u16)(d[r / 2] >> (r % 2 * 16)), to, r < n ? off + 2 * r : NOTHING, 0, 0);
  }
}

// Borders: in front of every (1 << every)-th block, where the last block begins (the gradient that comes in behind a sequence may
// be far larger than what is left of it a block earlier) and behind it.
DEV i64 borders_of(int nall, int every) { return ((nall - 1) >> every) + 3; }
DEV bool is_border(int c, int nreal, int every) { return (c & ((1 << every) - 1)) == 0 || c + 1 >= nreal; }
DEV i64 border_at(int c, int nreal, int nall, int every) {
  const int n = ((nall - 1) >> every) + 1;
  return c == nreal ? n : c + 1 == nreal ? n + 1 : c >> every;
}

// ================================================================== the walk over a sequence's blocks
#ifdef KERNEL_BLOCK
// One workgroup walks the blocks of one (batch, head, segment) for 64 of v's columns; wave w owns 16 of them: its share of
// the state, S^T [W x 16], stays in accumulators.  q and k are read by every workgroup of a head (up to four, on one XCD).
// A block: three waves form the 16 x 16 tiles of P on and below the diagonal; every wave adds the state's share of its
// columns of y, the block's own share, and updates its state.  The operands of blocks to come are on their way into
// registers meanwhile.
//
// What bounds it: latency.  With 8 x 1024 tokens x 32 heads of 128x128 in bfloat16, two workgroups per unit, a walk takes 105 us
// (its four tensors alone: 53 us at the rate of a large copy), and no pipe is near its limit: the vector pipes are busy 42 % of the
// time, the matrix cores 21 %, LDS 40 % (a third of that bank conflicts of the reads down columns), and waves wait for loads and
// barriers a third of theirs.  A block is four phases of one wave that follow each other, and two waves per SIMD hide each other
// only in part.  Blocks of 64 tokens took longer (P and its products grow with the block, and the tiles leave room for one
// workgroup), as did every other row stride in LDS; swapping pieces of rows instead has not been tried.
// With DOTS: dk 148 us (it also writes the states at borders, 84 MB), dq 158 us (it reads them), the state as three parts (24 of 58
// matrix products) and the sums in 64 bits.
//
// With DOTS the walk also leaves, per token, what the gradient of g is made of (see la_gate): forwards (dq) the products
// q_i.dq_i with the block's own share taken from unrounded numbers, less the share of each j; backwards (dk) the products
// k_j.dk_j of the state's share.  x is the operand of these products (q, k), in the 64 columns that the workgroup owns.  At
// borders between blocks the backward walk writes its state down, and the forward walk, which runs after it, multiplies its own
// with that.  Sums over column tiles are left to la_gate.  These sums are 64 bits: they are added up over many tokens.
struct Job {
  Tensor q, k, v, x;
  States init, fin;
  char* out;                // element (b, t, h, column): b * ob + t * ot + h / share * og + h % share * os + column
  i64 ob, ot, og, os, share, out_type;
  double* dots;             // [column tiles][B*H][T], or null: this job only goes along with one that has them
  float* marks;             // [B*H][borders][ceil(C/16)][W/16][64][4]: written backwards, read forwards
  double* inner;            // [B*H][borders][column tiles][4]: written forwards
  float* local;             // [B*H][nseg-1][column tiles][4][W/16][64][4]: states that segments leave behind, from zero
  double* totals;           // [B*H][nseg-1]: their sums of g
  i64 Hq, Hk, Hv, Hx;       // heads of the operands
  i64 width, C, back, pairs;      // q's and k's columns, v's columns, direction, whether dots take in P's share
  double in_scale, out_scale;     // of what enters the state (and P), of y
};
struct BlockArgs {
  Job job[2];
  Gate g;
  const i64* lengths;
  i64 B, T, H, nseg, per, tiles, every;   // per: blocks per segment; tiles: most column tiles of a job; every: of borders
};

constexpr int NT = W / 16, LT = 2;
constexpr int SPARTS = DOTS ? 3 : PP, SLIM = SPARTS - 1;
constexpr int QB = RP == 1 ? (W < 128 ? W / 32 : 4) : RP == 2 ? 2 : 1;       // operands read ahead: what 32 registers hold
constexpr int KB = RP == 1 ? 4 : RP == 2 ? 2 : 2;
constexpr bool EARLY = RP == 1 && W <= 128;                                  // registers for what dots need, ahead of its use
constexpr int SQ = stride_along(W), SK = stride_down(W), SV = stride_down(64), SX = stride_along(64), SP = stride_along(L);
constexpr int AT_K = OUT ? RP * L * SQ : 0, AT_V = AT_K + RP * L * SK, AT_X = AT_V + RP * L * SV, STAGE = AT_X + (DOTS ? RP * L * SX : 0);

template <int TYPE>
DEV void load_state(f4* S, const char* from, i64 at, i64 step, int rows, int g) {
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int row = 16 * nt + 4 * g + r;
      if (row < rows) S[nt][r] = load_type(from, at + row * step, TYPE);
    }
}
template <int TYPE>
DEV void store_state(const f4* S, float e, char* to, i64 at, i64 step, int rows, int g) {
#pragma unroll
  for (int nt = 0; nt < NT; nt++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int row = 16 * nt + 4 * g + r;
      if (row < rows) store_type(to, at + row * step, TYPE, S[nt][r] * e);
    }
}

DEV Frag<SPARTS> state_frag(const f4* S, int ks) {             // rows 32 ks + {4g..4g+3, 16+4g..16+4g+3} of a column
  const f4 u = S[2 * ks], v = S[2 * ks + 1];
  const float x[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
  return make_frag<SPARTS>(x);
}

extern "C" __global__ void __launch_bounds__(256, OCC) la_block(BlockArgs args) {
  __shared__ __attribute__((aligned(16))) u16 stage[NBUF][STAGE];
  __shared__ Decays decays[16];
#if OUT
  __shared__ __attribute__((aligned(16))) u16 P[NBUF][PP * L * SP];
#endif
#if !OUT
  __shared__ double totals[4];
#endif
#if DOTS
  __shared__ double of_rows[NBUF][LT][L], of_cols[NBUF][LT][L], of_state[NBUF][4][L];
#endif
  const Job& job = args.job[blockIdx.y];
  const int tid = threadIdx.x, lane = tid & 63, p = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int C = (int)job.C, ntiles = (C + 63) / 64;
  const i64 nseg = OUT ? args.nseg : args.nseg - 1;
  i64 group;
  int tile;
  if (!spread(blockIdx.x, (int)args.tiles, args.B * args.H * nseg, &group, &tile) || tile >= ntiles) return;
  const i64 bh = group / nseg, seg = group % nseg, b = bh / args.H, h = bh % args.H;
  const int c0 = tile * 64, cw = c0 + 16 * w, cols = C - c0 < 64 ? C - c0 : 64;
  const bool back = job.back != 0;
  const int T = (int)args.T, len = (int)length_of(args.lengths, b, T);
  const int nall = (T + L - 1) / L, nreal = (len + L - 1) / L;       // blocks; blocks with a token
  // this segment's steps: step o is block o, or nall - 1 - o backwards; those without a token only clear y
  const int s0 = (int)(seg * args.per), s1 = s0 + (int)args.per < nall ? s0 + (int)args.per : nall;
  const int first = back && s0 < nall - nreal ? (nall - nreal < s1 ? nall - nreal : s1) : s0;
  const int last = back || s1 < nreal ? s1 : (nreal > s0 ? nreal : s0);

  f4 S[NT];                 // column cw + p, rows 16 nt + 4 g + r
#pragma unroll
  for (int nt = 0; nt < NT; nt++) S[nt] = f4{0.f, 0.f, 0.f, 0.f};
#if OUT
  if (job.init.p) {
    const i64 at = b * job.init.sb + h * job.init.sh + (cw + p) * job.init.sc;
    const int rows = cw + p < C ? (int)job.width : 0;
    if (job.init.type == FP32) load_state<FP32>(S, job.init.p, at, job.init.sr, rows, g);
    else if (job.init.type == FP16) load_state<FP16>(S, job.init.p, at, job.init.sr, rows, g);
    else load_state<BF16>(S, job.init.p, at, job.init.sr, rows, g);
  }
#endif
#if OUT
#pragma unroll 4
  for (i64 s = 0; s < seg; s++) {                // the state at this segment's start
    const i64 at = bh * (nseg - 1) + s;
    const float e = expf((float)job.totals[at]);
    const f4* from = (const f4*)job.local + ((at * ntiles + tile) * 4 + w) * (NT * 64) + lane;
    for (int nt = 0; nt < NT; nt++) S[nt] = S[nt] * e + from[nt * 64];
  }
  for (int i = tid; i < NBUF * PP * L * SP / 8; i += 256) *(v4u*)(&P[0][0] + 8 * i) = v4u{0, 0, 0, 0};     // (stays zero above the diagonal)
#endif
#if DOTS
  if (tid < NBUF * LT * L) (&of_rows[0][0][0])[tid] = (&of_cols[0][0][0])[tid] = 0.0;
  // the border in front of block c (behind the last one: c = nreal), of those that count
  const int every = (int)args.every;
  const i64 borders = borders_of(nall, every);
  const auto counts = [&](int c) { return job.dots && c > 0 && c <= nreal && is_border(c, nreal, every); };
  const auto mark_of = [&](int c) {
    return (f4*)job.marks + ((bh * borders + border_at(c, nreal, nall, every)) * ((C + 15) / 16) + cw / 16) * (NT * 64) + lane;
  };
  f4 mark[NT];              // the backward walk's at this block's end, on its way while the block is worked on
  const auto mark_down = [&](int c) {
    if (!counts(c) || cw >= C) return;
    f4* at = mark_of(c);
    for (int nt = 0; nt < NT; nt++) at[nt * 64] = S[nt];
  };
  const auto mark_ahead = [&](int c) {
    if (!counts(c) || cw >= C) return;
    const f4* at = mark_of(c);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) mark[nt] = at[nt * 64];
  };
  // before the block in front of the border adds what is its own to the state, which it decays by `all`
  const auto mark_product = [&](int c, float all) {
    if (!counts(c)) return;
    if (!EARLY) mark_ahead(c);
    double s = 0.0;
    if (cw < C) {
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
        s += (double)(mark[nt][0] * S[nt][0] + mark[nt][1] * S[nt][1]) + (double)(mark[nt][2] * S[nt][2] + mark[nt][3] * S[nt][3]);
    }
    s = read_lane(scan64(s), 63) * all;
    if (lane == 0) job.inner[((bh * borders + border_at(c, nreal, nall, every)) * ntiles + tile) * 4 + w] = s;
  };
#endif

  const float in_scale = (float)job.in_scale;
  // a block o's operands, from the first block that this segment has
  const auto block_of = [&](int o) { return back ? nall - 1 - o : o; };
  const auto start = [&](auto& r, const Tensor& t, i64 heads, int col, int n) {
    r.init(t, t.p + (b * t.sb + h / (args.H / heads) * t.sh + (i64)block_of(first) * L * t.st + col * t.sn) * ESZ, n, back, tid);
  };
  Staging<W, SK> rk;
  Staging<64, SV> rv;
  start(rk, job.k, job.Hk, 0, (int)job.width);
  start(rv, job.v, job.Hv, c0, cols);
#if OUT
  Staging<W, SQ> rq;
  start(rq, job.q, job.Hq, 0, (int)job.width);
#endif
#if DOTS
  Staging<64, SX> rx;
  start(rx, job.x, job.Hx, c0, job.dots ? cols : 0);
#endif
  // (always a block further; behind the last one nothing is read)
  const auto fetch = [&](int o) {
    const int tokens = o < last ? len - block_of(o) * L : 0;
#if OUT
    rq.load(tokens);
#endif
    rk.load(tokens);
    rv.load(tokens);
#if DOTS
    rx.load(tokens);
#endif
  };
  const auto put = [&](u16* to) {
#if OUT
    rq.store(to, tid);
#endif
    rk.store(to + AT_K, tid);
    rv.store(to + AT_V, tid);
#if DOTS
    rx.store(to + AT_X, tid);
#endif
  };
  // Decays are prepared for eight blocks at a time, two by each wave (a block per half); backwards a row's gate is the one
  // of the token behind it.  `rg`: the gates of the eight blocks after those.
  const auto gates = [&](int o) {
    const int i = lane & (L - 1);
    o += 2 * w + lane / L;
    const int t = block_of(o) * L + (back ? L - i : i);
    return o < last && t < len ? raw_gate(args.g, b, h, t) : 0u;         // (zero is 0.0 in every type)
  };
  double total = 0.0;
  const auto fill = [&](int o, u32 raw) {
    const int at = (o - first + 2 * w) & 15;
    total += fill_decays(decays + at, decays + at + 1, gate_value(args.g, raw), in_scale, lane);
  };
  u32 rg = 0;
  if (first < last) {
    fetch(first);
    const u32 now = gates(first);
    rg = gates(first + 8);
    fill(first, now);
    put(stage[0]);
    if constexpr (NBUF == 2) {
      fetch(first + 1);
      put(stage[1]);
    }
  }
  __syncthreads();
#if OUT
  const float out_scale = (float)job.out_scale;
  const bool wide = FAST ? WIDE != 0 : job.out_type == FP32;       // (or of the operands' type)
  const bool whole = FAST || C % 4 == 0;
  const int size = wide ? 4 : ESZ;
  const i64 out_at = b * job.ob + h / job.share * job.og + h % job.share * job.os;
  char* to = job.out + (out_at + (i64)block_of(first) * L * job.ot) * size;
  const i64 to_step = (back ? -L : L) * job.ot * size;
  u32 to_off[LT];
#pragma unroll
  for (int i = 0; i < LT; i++) to_off[i] = (u32)((back ? L - 1 - (16 * i + p) : 16 * i + p) * job.ot + cw + 4 * g) * size;

  // waves 0..2 each form a tile of P: column pi, rows pj..pj+3 (wave 3 goes along and keeps nothing)
  const int it = w > 0, jt = w > 1, pi = 16 * it + p, pj = 16 * jt + 4 * g;
  struct Pair {
    f4 apart;
    Frag<RP> kj[QB], qi[QB];
#if DOTS
    Frag<RP> vj[2], xi[2];
#endif
  };
  const auto pair_operands = [&](Pair& x, const u16* tiles, int k0) {
#pragma unroll
    for (int ks = 0; ks < QB; ks++) {
      x.kj[ks] = along8<SK>(tiles + AT_K, 16 * jt + p, 32 * (k0 + ks), g);
      x.qi[ks] = along8<SQ>(tiles, pi, 32 * (k0 + ks), g);
    }
  };
#if DOTS
  const auto own_operands = [&](Pair& x, const u16* tiles) {
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      x.vj[ks] = along8<SV>(tiles + AT_V, 16 * jt + p, 32 * ks, g);
      x.xi[ks] = along8<SX>(tiles + AT_X, pi, 32 * ks, g);
    }
  };
#endif
  const auto pair_begin = [&](Pair& x, const u16* tiles, const Decays& D) {
    x.apart = (D.hi[pi] - *(const f4*)(D.hi + pj)) + (D.lo[pi] - *(const f4*)(D.lo + pj));
    pair_operands(x, tiles, 0);
#if DOTS
    if (EARLY) own_operands(x, tiles);
#endif
  };
  const auto pair_product = [&](Pair& x, const u16* tiles) {
    f4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k0 = 0; k0 < W / 32; k0 += QB) {
      if (k0 > 0) pair_operands(x, tiles, k0);
#pragma unroll
      for (int ks = 0; ks < QB; ks++) c = mul<RAW>(x.kj[ks], x.qi[ks], c);
    }
    return c;
  };
  const auto pair_end = [&](Pair& x, f4 c, const u16* tiles, int o) {
#pragma unroll
    for (int r = 0; r < 4; r++) c[r] = pj + r <= pi ? c[r] * (__builtin_amdgcn_exp2f(x.apart[r]) * in_scale) : 0.f;
    u32 d[PP * 2];
    split2<PP>(c[0], c[1], d, 2);
    split2<PP>(c[2], c[3], d + 1, 2);
    if (w < 3) {
#pragma unroll
      for (int q = 0; q < PP; q++) *(v2u*)(P[o % NBUF] + (q * L + pi) * SP + pj) = v2u{d[2 * q], d[2 * q + 1]};
    }
#if DOTS
    if (job.pairs && w < 3) {
      f4 a = {0.f, 0.f, 0.f, 0.f};
      if (!EARLY) own_operands(x, tiles);
#pragma unroll
      for (int ks = 0; ks < 2; ks++) a = mul<RAW>(x.vj[ks], x.xi[ks], a);
      double row = 0.0;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const double s = pj + r <= pi ? (double)(c[r] * a[r]) : 0.0;       // (a need not be finite where c is zero)
        row += s;
        const double col = row_of_16(s);
        if (p == 15) of_cols[o % NBUF][it][pj + r] = col;
      }
      row = over_rows(row);
      if (g == 3) of_rows[o % NBUF][jt][pi] = row;
    }
#endif
  };
  f4 y[LT];                                      // column i = 16 it + p, rows cw + 4 g + r
  Frag<RP> vf = {};
  bool odd = false;                              // whether a lane of this wave has an infinity or a NaN in it
  const auto own_share = [&](int n) {            // of block n, whose P lies in LDS
    const u16* own = P[n % NBUF];
    const Frag<PP> p0 = along<SP, PP>(own, p, 0, g), p1 = along<SP, PP>(own, 16 + p, 0, g);
    int from = L;                                // row of the first infinity or NaN in column cw + p
    if (odd) {
      // The zeros of P above its diagonal must not meet them (an earlier token would be NaN): they come out of the factor, and
      // their column is NaN from the first of them on, as the state is from the next block on.  Looking for them takes 1 to 2 %
      // of the time; all of this stands here because a branch in the middle of a block cost 50 registers.
      float x[8];
      frag_values(vf, x);
      for (int e = 0; e < 8; e++) {
        if (__builtin_isfinite(x[e])) continue;
        const int row = (e / 4) * 16 + 4 * g + e % 4;
        from = row < from ? row : from;
        for (int q = 0; q < RP; q++) vf.d[q][e / 2] &= e % 2 ? 0xffffu : 0xffff0000u;
      }
      for (int far = 16; far < 64; far *= 2) {
        const int other = __shfl_xor(from, far);
        from = other < from ? other : from;
      }
    }
    y[0] = mul<PP - 1>(vf, p0, y[0]);
    y[1] = mul<PP - 1>(vf, p1, y[1]);
    if (odd) {
      for (int r = 0; r < 4; r++) {
        const int row = __shfl(from, 4 * g + r);
        for (int i = 0; i < LT; i++) y[i][r] = 16 * i + p < row ? y[i][r] : __builtin_nanf("");
      }
    }
  };
  const auto write = [&](int o, bool any) {
    const Buffer into = buffer_at(to);
    if (any) to += to_step;
#pragma unroll
    for (int it = 0; it < LT; it++) {
      const int i = back ? L - 1 - (16 * it + p) : 16 * it + p;
      const int t0 = block_of(o) * L;
      const f4 z = t0 + i < len ? y[it] * out_scale : f4{0.f, 0.f, 0.f, 0.f};
      const u32 off = any && t0 + i < T ? to_off[it] : NOTHING;
      if (wide) store_wide(into, off, z, C - cw - 4 * g, whole);
      else store_in(into, off, z, C - cw - 4 * g, whole);
    }
  };
#pragma unroll
  for (int i = 0; i < LT; i++) y[i] = f4{0.f, 0.f, 0.f, 0.f};
#endif
#if DOTS
  if (back && first < last && block_of(first) == nreal - 1) mark_down(nreal);
#endif
  for (int o = first; o < last; o++) {
    // With two tiles in LDS, the block's own share of y is added a block later: one barrier a block stands between P's writers
    // and its readers, and between a tile's readers and its next writers.  (P a block ahead,
    // which needs two, is 2 to 5 % slower.)
    const int n = o - first;
    const u16* tiles = stage[n % NBUF];
    const u16 *K = tiles + AT_K, *V = tiles + AT_V;
    const Decays& D = decays[n & 15];
    fetch(o + NBUF);
#if DOTS
    if (EARLY && !back) mark_ahead(o + 1);
#endif
    // What a block needs is read from LDS well ahead of its use, and the parts of the decayed v fill the wait.  (The
    // compiler's own order within that: scheduling fences that kept this one made a block 5 % slower.)
    const float all = D.from_start[L - 1];
    const f4 to0 = *(const f4*)(D.to_end + 4 * g), to1 = *(const f4*)(D.to_end + 16 + 4 * g);
#if OUT
    if constexpr (NBUF == 2) {
      own_share(n + 1);                          // (the one before: two are kept)
      write(o - 1, n > 0);
    }
    vf = down<SV>(V, 0, 16 * w, lane);
    const u16* Q = tiles;
    const float from[LT] = {D.from_start[p], D.from_start[16 + p]};
    Pair pair;
    pair_begin(pair, tiles, D);
    Frag<RP> qf[QB][LT];
#pragma unroll
    for (int x = 0; x < QB; x++)
#pragma unroll
      for (int i = 0; i < LT; i++) qf[x][i] = along<SQ>(Q, 16 * i + p, 32 * x, g);
#else
    const Frag<RP> vf = down<SV>(V, 0, 16 * w, lane);
#endif
    float vx[8];
    frag_values(vf, vx);
#if OUT
    const float sum = (fabsf(vx[0]) + fabsf(vx[1])) + (fabsf(vx[2]) + fabsf(vx[3])) + ((fabsf(vx[4]) + fabsf(vx[5])) + (fabsf(vx[6]) + fabsf(vx[7])));
    odd = __any(!__builtin_isfinite(sum));
#endif
#pragma unroll
    for (int r = 0; r < 4; r++) {
      vx[r] *= to0[r];
      vx[4 + r] *= to1[r];
    }
    const Frag<3> vd = make_frag<3>(vx);
#if OUT
#pragma unroll
    for (int i = 0; i < LT; i++) y[i] = f4{0.f, 0.f, 0.f, 0.f};
    const f4 product = pair_product(pair, tiles);
#endif
    Frag<RP> kf[KB];
#pragma unroll
    for (int x = 0; x < KB; x++) kf[x] = down<SK>(K, 0, 16 * x, lane);
#if OUT
#pragma unroll
    for (int k0 = 0; k0 < W / 32; k0 += QB) {
#pragma unroll
      for (int ks = 0; ks < QB; ks++) {
        const Frag<SPARTS> s = state_frag(S, k0 + ks);
#pragma unroll
        for (int i = 0; i < LT; i++) y[i] = mul<SLIM>(s, qf[ks][i], y[i]);
      }
      if (k0 + QB < W / 32) {
#pragma unroll
        for (int x = 0; x < QB; x++)
#pragma unroll
          for (int i = 0; i < LT; i++) qf[x][i] = along<SQ>(Q, 16 * i + p, 32 * (k0 + QB + x), g);
      }
    }
    pair_end(pair, product, tiles, n);
#pragma unroll
    for (int i = 0; i < LT; i++) y[i] *= from[i];
#if DOTS
#pragma unroll
    for (int i = 0; i < LT; i++) {
      double s = 0.0;
#pragma unroll
      for (int q = 0; q < RP; q++) {
        const v2u x = *(const v2u*)(tiles + AT_X + (q * L + 16 * i + p) * SX + 16 * w + 4 * g);
        s += (double)y[i][0] * (double)as_f(x[0] << 16) + (double)y[i][1] * (double)as_f(x[0] & 0xffff0000u);
        s += (double)y[i][2] * (double)as_f(x[1] << 16) + (double)y[i][3] * (double)as_f(x[1] & 0xffff0000u);
      }
      s = over_rows(s);
      if (g == 3) of_state[n % NBUF][w][16 * i + p] = s;
    }
#endif
#endif
#if DOTS
    if (!back) mark_product(o + 1, all);
#endif
#pragma unroll
    for (int n0 = 0; n0 < NT; n0 += KB) {
      Frag<RP> next[KB];
      if (n0 + KB < NT) {
#pragma unroll
        for (int x = 0; x < KB; x++) next[x] = down<SK>(K, 0, 16 * (n0 + KB + x), lane);
      }
#pragma unroll
      for (int x = 0; x < KB; x++) S[n0 + x] *= all;
      mul_each<KB, 2>(kf, vd, S + n0);
      if (n0 + KB < NT) {
#pragma unroll
        for (int x = 0; x < KB; x++) kf[x] = next[x];
      }
    }
#if OUT
    if constexpr (NBUF == 1) {
      __syncthreads();
      own_share(n);
    }
#endif
    if ((n & 7) == 6) {
      fill(o + 2, rg);
      rg = gates(o + 10);
    }
    if constexpr (NBUF == 2 || !OUT) __syncthreads();        // (everybody is done with this block's tile)
    put(stage[n % NBUF]);
#if DOTS
    if (w == 3 && lane < L) {
      const int t = block_of(o) * L + (back ? L - 1 - lane : lane);
      const auto& of = of_state[n % NBUF];
      double s = of[0][lane] + of[1][lane] + (of[2][lane] + of[3][lane]);
      if (job.pairs) s += (of_rows[n % NBUF][0][lane] + of_rows[n % NBUF][1][lane]) - (of_cols[n % NBUF][0][lane] + of_cols[n % NBUF][1][lane]);
      if (job.dots && t < T) job.dots[((i64)tile * args.B * args.H + bh) * T + t] = s * job.out_scale;
    }
    if (back) mark_down(block_of(o));
#endif
#if OUT
    if constexpr (NBUF == 1) write(o, true);
#endif
    if constexpr (NBUF == 1) __syncthreads();
  }
#if OUT
  if constexpr (NBUF == 2) {
    if (first < last) {
      own_share(last - 1 - first);
      write(last - 1, true);
    }
  }
  for (int o = s0; o < s1; o++) {                // blocks without a token
    if (o >= first && o < last) continue;
    for (int u = tid; u < L * 16; u += 256) {
      const int t = block_of(o) * L + u / 16;
      const int col = c0 + u % 16 * 4;
      if (t < T)
        for (int r = 0; r < 4 && col + r < C; r++) store_type(job.out, out_at + t * job.ot + col + r, wide ? FP32 : IN, 0.f);
    }
  }
  if (job.fin.p && seg == nseg - 1) {
    const float e = back && len > 0 ? expf((float)gate_of(args.g, b, h, 0)) : 1.f;
    int mine = p;
    asm("" : "+v"(mine));                        // (or the addresses of the first state stay in registers all the while)
    const i64 at = b * job.fin.sb + h * job.fin.sh + (cw + mine) * job.fin.sc;
    const int rows = cw + mine < C ? (int)job.width : 0;
    if (job.fin.type == FP32) store_state<FP32>(S, e, job.fin.p, at, job.fin.sr, rows, g);
    else if (job.fin.type == FP16) store_state<FP16>(S, e, job.fin.p, at, job.fin.sr, rows, g);
    else store_state<BF16>(S, e, job.fin.p, at, job.fin.sr, rows, g);
  }
#else
  const i64 at = bh * (args.nseg - 1) + seg;
  f4* to = (f4*)job.local + ((at * ntiles + tile) * 4 + w) * (NT * 64) + lane;
  for (int nt = 0; nt < NT; nt++) to[nt * 64] = S[nt];
  if (lane == 0) totals[w] = total;
  __syncthreads();
  if (tid == 0 && tile == 0) job.totals[at] = totals[0] + totals[1] + (totals[2] + totals[3]);
#endif
}
#endif

// ================================================================== gradient of the decays
#ifdef KERNEL_GATE
// The gradient of g_t is what token t's step carries over, <X, exp(g_t) S>.  For the tokens of a block that ends at a border the
// walks left the product of X behind it with the state in front of it, decayed through the block; that and
//     sum over i >= t of q_i.dq_i  +  sum over j < t of k_j.dk_j                (i, j in the block)
// is the result, sums of terms that exp(g_t) is part of: with a fast decay, or an empty state, nothing larger has to cancel.
// From the first token of a block to the block before, and from one token to the one before it in blocks without a border,
//     <X, S> + q_t.dq_t - k_t.dk_t.
// Summed backwards in 64 bits from the nearest border, never over a whole sequence, where what is left of a fast decay would drown
// in the rounding of what came before.  Borders stand every eight blocks; at every block where all tokens share a decay, whose gradient
// counts a token's error once for each token in front of it in the span (3 x 4877 tokens, one head, float32, terms that cancel to
// 1/300: 3e-5 off with eight blocks, 6e-6 with two, 1e-6 with one; a training step of 8 x 1024 tokens x 32 heads of 128x128 takes
// 489, 531 and 620 us).  The tokens' products come in 64 bits, too: their rounding to 32 was the largest error of all.  The block's
// own share of q.dq and k.dk is the same numbers once by rows and once by columns, so it cancels where it should.
// One workgroup per (batch, head, 32 blocks), a token per thread, a block per half wave.  Bound by waiting for its few loads: 10 us
// for 8 x 1024 tokens x 32 heads (25 MB).
struct GateArgs {
  const double* dots_q;     // [tiles][B*H][T]
  const double* dots_k;
  const double* inner;      // [B*H][borders][parts]
  Gate g;
  char* dg;                 // [B,T,H]
  const i64* lengths;
  i64 B, T, H, tiles, type, init, every;      // init: whether there is a state in front of the first token
};

extern "C" __global__ void __launch_bounds__(1024) la_gate(GateArgs a) {
  __shared__ double sums_q[32], sums_k[32], ends[33];     // a block's; what a border in front of a block (or none: unused) holds
  const int tid = threadIdx.x, lane = tid & 63, blk = tid / L;
  const int T = (int)a.T, nall = (T + L - 1) / L, groups = (nall + 31) / 32;
  const i64 bh = blockIdx.x / groups, b = bh / a.H, h = bh % a.H, BH = a.B * a.H;
  const int c0 = (int)(blockIdx.x % groups) * 32, c = c0 + blk;
  const int len = (int)length_of(a.lengths, b, T), nreal = (len + L - 1) / L, parts = 4 * (int)a.tiles, every = (int)a.every;
  if (tid < 33) {
    const int at = c0 + tid;
    double x = 0.0;
    if (at > 0 && at <= nreal && is_border(at, nreal, every)) {
      const double* from = a.inner + (bh * borders_of(nall, every) + border_at(at, nreal, nall, every)) * parts;
      for (int i = 0; i < parts; i++) x += from[i];
      if (at < nreal) x *= exp(gate_of(a.g, b, h, (i64)at * L));         // (inside the sequence the walk has yet to decay by it)
    }
    ends[tid] = x;
  }
  // half a wave holds a block back to front
  const int t = c * L + L - 1 - (tid & (L - 1));
  double dq = 0.0, dk = 0.0;
  if (t < len)
    for (i64 k = 0; k < a.tiles; k++) {
      dq += a.dots_q[(k * BH + bh) * T + t];
      dk += a.dots_k[(k * BH + bh) * T + t];
    }
  dq = scan32(dq);
  dk = scan32(dk);
  if ((lane & (L - 1)) == L - 1) {
    sums_q[blk] = dq;
    sums_k[blk] = dk;
  }
  __syncthreads();
  if (t >= T) return;
  double x = 0.0;
  // (a decay of zero carries nothing over: what the sums around it leave is rounding)
  if (t < len && (t > 0 || a.init) && !(gate_of(a.g, b, h, t) <= ZERO_DECAY)) {
    x = dq;
    int at = blk + 1;
    if (is_border(c0 + at, nreal, every)) x += sums_k[blk] - dk;
    else {
      x -= dk;
      for (; !is_border(c0 + at + 1, nreal, every); at++) x += sums_q[at] - sums_k[at];       // (32 blocks on is a border)
      x += sums_q[at++];
    }
    x += ends[at];
  }
  store_type(a.dg, (b * a.T + t) * a.H + h, (int)a.type, (float)x);
}
#endif

// ================================================================== one token
#ifdef KERNEL_STEP
// S = exp(g) S + v k^T in place, y = scale S q.  Bound by reading and writing the state once: 111 us for 128 sequences x
// 32 heads of 128x128 in fp32 and 27 us for 256 x 32 heads of 64x64 in bfloat16 (4.9 and 5.0 TB/s of the 5.1 that a large copy
// reaches), 8 us for one sequence, which is the call.  A wave takes some rows of one head, so that small heads fill a workgroup
// too (a workgroup per head: 37 us in the second case).  A group of `gl` lanes owns rows of the state, a lane VE neighbouring
// columns (16 bytes) of each, whose q and k it holds; R rows are in flight at a time.  States that do not allow 16-byte accesses
// go column by column.
struct StepArgs {
  Tensor q, k, v;           // st unused
  Gate g;
  States s;
  char* y;                  // [B,H,M]
  i64 B, H, Hk, M, N, vec, gl, rows;      // rows of the state per wave
  double scale;
};
DEV float load_in(const char* p, i64 i) { return load_type(p, i, IN); }

template <int TYPE>
DEV void unpack(const v4u t, float* s) {
  if constexpr (TYPE == FP32) {
    for (int i = 0; i < 4; i++) s[i] = as_f(t[i]);
  } else {
    for (int i = 0; i < 8; i++) {
      const u16 x = (u16)(t[i / 2] >> (i % 2 * 16));
      s[i] = TYPE == FP16 ? half_to_f(x) : as_f((u32)x << 16);
    }
  }
}
template <int TYPE>
DEV v4u pack(const float* s) {
  v4u t;
  for (int i = 0; i < 4; i++) {
    if constexpr (TYPE == FP32) t[i] = as_u(s[i]);
    else if constexpr (TYPE == BF16) t[i] = pack_rne(s[2 * i], s[2 * i + 1]);
    else t[i] = (u32)__builtin_bit_cast(u16, (_Float16)s[2 * i]) | (u32)__builtin_bit_cast(u16, (_Float16)s[2 * i + 1]) << 16;
  }
  return t;
}

struct Token {              // one head's operands
  const char *q, *k, *v;
  char *s, *y;
  float e, scale;
};

template <int TYPE>
DEV void step_rows(const StepArgs& a, const Token& t, int r0, int end, int lane) {
  constexpr int VE = TYPE == FP32 ? 4 : 8, SZ = 16 / VE, R = 4;
  const int gl = (int)a.gl, sub = lane % gl, grp = lane / gl, groups = 64 / gl, N = (int)a.N, n = sub * VE;
  float q[VE], k[VE];
  for (int i = 0; i < VE; i++) {
    q[i] = n < N ? load_in(t.q, (n + i) * a.q.sn) * t.scale : 0.f;
    k[i] = n < N ? load_in(t.k, (n + i) * a.k.sn) : 0.f;
  }
  char* at = t.s + (i64)n * SZ;
  for (int m0 = r0; m0 < end; m0 += groups * R) {
    v4u raw[R];
    float v[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int m = m0 + i * groups + grp;
      const bool in = m < end && n < N;
      raw[i] = in ? *(const v4u*)(at + m * a.s.sr * SZ) : v4u{0, 0, 0, 0};
      v[i] = m < end ? load_in(t.v, m * a.v.sn) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
      const int m = m0 + i * groups + grp;
      float s[VE], acc = 0.f;
      unpack<TYPE>(raw[i], s);
      for (int x = 0; x < VE; x++) {
        s[x] = t.e * s[x] + v[i] * k[x];
        acc += s[x] * q[x];
      }
      if (m < end && n < N) *(v4u*)(at + m * a.s.sr * SZ) = pack<TYPE>(s);
      acc = sum_lanes(acc, gl);
      if (m < end && sub == 0) store_type(t.y, m, IN, acc);
    }
  }
}

DEV void step_columns(const StepArgs& a, const Token& t, int r0, int end, int lane) {
  const int gl = (int)a.gl, sub = lane % gl, grp = lane / gl, groups = 64 / gl, type = (int)a.s.type;
  for (int m0 = r0; m0 < end; m0 += groups) {
    const int m = m0 + grp;
    float acc = 0.f;
    if (m < end) {
      const float v = load_in(t.v, m * a.v.sn);
      for (int n = sub; n < a.N; n += gl) {
        const i64 i = m * a.s.sr + n * a.s.sc;
        const float s = t.e * load_type(t.s, i, type) + v * load_in(t.k, n * a.k.sn);
        acc += s * load_in(t.q, n * a.q.sn) * t.scale;
        store_type(t.s, i, type, s);
      }
    }
    acc = sum_lanes(acc, gl);
    if (m < end && sub == 0) store_type(t.y, m, IN, acc);
  }
}

extern "C" __global__ void __launch_bounds__(256) la_step(StepArgs a) {
  const u32 unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per = (u32)((a.M + a.rows - 1) / a.rows), bh = unit / per;
  if (bh >= a.B * a.H) return;
  const i64 b = bh / (u32)a.H, h = bh % (u32)a.H, hk = h / (a.H / a.Hk);
  const int r0 = (int)(unit % per * a.rows), end = r0 + (int)a.rows < a.M ? r0 + (int)a.rows : (int)a.M, lane = threadIdx.x & 63;
  Token t;
  t.q = a.q.p + (b * a.q.sb + hk * a.q.sh) * ESZ;
  t.k = a.k.p + (b * a.k.sb + hk * a.k.sh) * ESZ;
  t.v = a.v.p + (b * a.v.sb + h * a.v.sh) * ESZ;
  t.s = a.s.p + (b * a.s.sb + h * a.s.sh) * (a.s.type == FP32 ? 4 : 2);
  t.y = a.y + (i64)bh * a.M * ESZ;
  t.e = expf((float)gate_of(a.g, b, h, 0));
  t.scale = (float)a.scale;
  if (!a.vec) step_columns(a, t, r0, end, lane);
  else if (a.s.type == FP32) step_rows<FP32>(a, t, r0, end, lane);
  else if (a.s.type == BF16) step_rows<BF16>(a, t, r0, end, lane);
  else step_rows<FP16>(a, t, r0, end, lane);
}
#endif
