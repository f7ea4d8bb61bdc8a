// Layer norm over the last axis, forward and backward (gfx950).
//
//     y = xhat * w + b,   xhat = (x - mean) * rstd,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//     d = dy * w:         dx = rstd * (d - mean(d) - xhat * mean(d * xhat)),   dw = sum dy * xhat,   db = sum dy
//
// w and b belong to a column, or to a head and a column (row r uses row r % heads of them).
//
// Bound by memory: x is read and y written once; backward reads x and dy and writes dx.  Mean and rstd are formed again
// from the row that the backward pass holds anyway, so the forward pass saves nothing but x.  A row lives in the registers
// of a team: GL lanes of a wave (a power of two; 64 / GL rows side by side in a wave) with K pieces of 16 bytes each, or,
// where a wave's registers do not hold a row (WIDE), the whole workgroup.  Teams walk the rows in steps that are a
// multiple of `heads`, so a team's w and b - and its share of dw and db - stay in registers, and the next row's loads are
// issued before the current row is worked on.  Shares of dw and db meet in two steps in a fixed order (per team in fp32,
// between teams by the kernel that sums slices in 64 bits), never in atomics.
//
// Measured against the 5.1 TB/s of a large copy, per-column w and b in fp32: forward 8192 x 4096 bfloat16 32 us (4.2 TB/s),
// 262144 x 128 27 us (5.0), 2048 x 16384 39 us (3.4), 4096 x 8192 float32 46 us (5.8, part of it from the last-level cache);
// forward and backward together 95, 97, 151 and 148 us (five passes of 67 or 134 MB: 3.5, 3.5, 2.2 and 4.5 TB/s).  Backward, the
// registers for w, dw and db leave fewer rows in flight, and 1024 threads (over 8192 columns) spill some of them.
//
// Sums over a row are fp32 and two passes over registers (mean first, then squares of what is left): no cancellation.
//
// Compiled by flex_rnn_amd/handwritten.py with IN (0 bfloat16, 1 float16, 2 float32), K, TH (threads), GL, WIDE and BACKWARD.
#include <hip/hip_runtime.h>

typedef unsigned int u32;
typedef unsigned short u16;
typedef long long i64;
typedef __bf16 bh2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef u32 v4u __attribute__((ext_vector_type(4)));

#define DEV static __device__ __forceinline__

enum { BF16 = 0, FP16 = 1, FP32 = 2 };
constexpr int ESZ = IN == FP32 ? 4 : 2;
constexpr int VE = 16 / ESZ;

struct Args {
  const char* x;            // row r = (outer, head): outer * sx + head * hx elements, then C next to each other
  const char* dy;
  char* y;                  // forward: y; backward: dx; [rows, C] without gaps
  const char *w, *b;        // [heads, C] or null
  float *dw, *db;           // backward: [teams / heads][heads][C] or null
  i64 rows, heads, C, sx, hx, sy, hy, w_type, b_type, vec, teams;
  double eps;
};

DEV float as_f(u32 x) { return __uint_as_float(x); }
DEV float half_to_f(u16 h) { return (float)__builtin_bit_cast(_Float16, h); }
DEV u32 pack_bf16(float a, float b) {
  f2 v = {a, b};
  return __builtin_bit_cast(u32, __builtin_convertvector(v, bh2));
}
DEV float load_type(const char* p, i64 i, int type) {
  if (type == FP32) return ((const float*)p)[i];
  const u16 h = ((const u16*)p)[i];
  return type == FP16 ? half_to_f(h) : as_f((u32)h << 16);
}

struct Piece {               // 16 bytes of a row as they are in memory
  v4u d;
};

// 16 bytes at any address of the element type
typedef v4u v4u_any __attribute__((aligned(2)));

// Columns start .. start + VE - 1 of a row.  A row's last piece is moved back so that it ends with the row: its first `skip`
// columns belong to the piece before it too, are left out of sums, and come out the same twice.  (Whole pieces at any address:
// 33588 rows of 999 bfloat16 take 30 us, 91 one element at a time.)  Of a row shorter than a piece, `start` is negative.
DEV Piece load_piece(const char* row, int start, int skip, bool vec) {
  Piece r;
  r.d = v4u{0, 0, 0, 0};
  if (vec) {
    if (skip < VE) r.d = *(const v4u_any*)(row + (i64)start * ESZ);
  } else {
    for (int e = 0; e < VE; e++)
      if (e >= skip) {
        if constexpr (IN == FP32) r.d[e] = ((const u32*)row)[start + e];
        else r.d[e / 2] |= (u32)((const u16*)row)[start + e] << (e % 2 * 16);
      }
  }
  return r;
}
DEV void values(const Piece& r, float* x) {
  for (int e = 0; e < VE; e++) {
    if constexpr (IN == FP32) x[e] = as_f(r.d[e]);
    else if constexpr (IN == FP16) x[e] = half_to_f((u16)(r.d[e / 2] >> (e % 2 * 16)));
    else x[e] = e % 2 ? as_f(r.d[e / 2] & 0xffff0000u) : as_f(r.d[e / 2] << 16);
  }
}
DEV void store_piece(char* row, int start, int skip, bool vec, const float* x) {
  v4u d;
  for (int e = 0; e < 4; e++) {
    if constexpr (IN == FP32) d[e] = __float_as_uint(x[e]);
    else if constexpr (IN == BF16) d[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
    else d[e] = (u32)__builtin_bit_cast(u16, (_Float16)x[2 * e]) | (u32)__builtin_bit_cast(u16, (_Float16)x[2 * e + 1]) << 16;
  }
  if (vec) {
    if (skip < VE) *(v4u_any*)(row + (i64)start * ESZ) = d;
  } else {
    for (int e = 0; e < VE; e++)
      if (e >= skip) {
        if constexpr (IN == FP32) ((u32*)row)[start + e] = d[e];
        else ((u16*)row)[start + e] = (u16)(d[e / 2] >> (e % 2 * 16));
      }
  }
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
DEV float sum_lanes(float x, int lanes) {      // over groups of 1 to 64 lanes, a power of two (the same in a whole wave)
  if (lanes >= 2) x = sum2(x);
  if (lanes >= 4) x = dpp_add<0x4e>(x);
  if (lanes >= 8) x = dpp_add<0x141>(x);
  if (lanes >= 16) x = dpp_add<0x140>(x);
  if (lanes >= 32) x = sum_rows16(x);
  if (lanes >= 64) x = sum_rows32(x);
  return x;
}

// sums of two numbers over a team, known to all its lanes afterwards
DEV f2 team_sum(f2 s, int gl, float (*lds)[2], int tid) {
  s[0] = sum_lanes(s[0], gl);
  s[1] = sum_lanes(s[1], gl);
#if WIDE
  __syncthreads();
  if ((tid & 63) == 0) {
    lds[tid >> 6][0] = s[0];
    lds[tid >> 6][1] = s[1];
  }
  __syncthreads();
  s = f2{0.f, 0.f};
  for (int i = 0; i < TH / 64; i++) {
    s[0] += lds[i][0];
    s[1] += lds[i][1];
  }
#endif
  return s;
}

extern "C" __global__ void __launch_bounds__(TH)
#if BACKWARD
ln_bw(Args a) {
#else
ln_fw(Args a) {
#endif
#if WIDE
  __shared__ float lds[TH / 64][2];
#else
  float (*lds)[2] = nullptr;
#endif
  const int tid = threadIdx.x, gl = WIDE ? 64 : GL;
  const int sub = WIDE ? tid : tid % gl, lanes = WIDE ? TH : gl;
  const i64 team = WIDE ? (i64)blockIdx.x : (i64)blockIdx.x * (TH / gl) + tid / gl;
  const int C = (int)a.C;
  const bool vec = a.vec != 0, live = team < a.teams;
  const i64 head = live ? team % a.heads : 0;
  const float inv = 1.f / (float)C, eps = (float)a.eps;

  int start[K], skip[K];
#pragma unroll
  for (int k = 0; k < K; k++) {
    const int n = (sub + k * lanes) * VE;
    start[k] = n < C - VE ? n : C - VE;
    skip[k] = n - start[k] < VE ? n - start[k] : VE;
  }
  float w[K * VE];
#if !BACKWARD
  float b[K * VE];
#endif
  for (int k = 0; k < K; k++)
    for (int e = 0; e < VE; e++) {
      const int n = start[k] + e;
      const bool in = n >= 0 && skip[k] < VE;
      w[k * VE + e] = a.w && in ? load_type(a.w, head * C + n, (int)a.w_type) : 1.f;
#if !BACKWARD
      b[k * VE + e] = a.b && in ? load_type(a.b, head * C + n, (int)a.b_type) : 0.f;
#endif
    }
#if BACKWARD
  float dw[K * VE], db[K * VE];
  for (int i = 0; i < K * VE; i++) dw[i] = db[i] = 0.f;
  Piece ny[K];
#endif
  Piece nx[K];
  const i64 step = a.teams / a.heads;            // outer rows between a team's rows
  const i64 outers = a.rows / a.heads;
  const auto fetch = [&](i64 o) {
#pragma unroll
    for (int k = 0; k < K; k++) {
      nx[k] = load_piece(a.x + (o * a.sx + head * a.hx) * ESZ, start[k], skip[k], vec);
#if BACKWARD
      ny[k] = load_piece(a.dy + (o * a.sy + head * a.hy) * ESZ, start[k], skip[k], vec);
#endif
    }
  };
  const i64 first = live ? team / a.heads : outers;
  if (first < outers) fetch(first);
  // (lanes of one wave may belong to teams with and without a row left: sums run over a team's own lanes only)
  for (i64 o = first; o < outers; o += step) {
    float x[K * VE];
#pragma unroll
    for (int k = 0; k < K; k++) values(nx[k], x + k * VE);
#if BACKWARD
    float d[K * VE];
#pragma unroll
    for (int k = 0; k < K; k++) values(ny[k], d + k * VE);
#endif
    if (o + step < outers) fetch(o + step);
    float s = 0.f;
    for (int i = 0; i < K * VE; i++) s += i % VE >= skip[i / VE] ? x[i] : 0.f;
    const float mean = team_sum(f2{s, 0.f}, gl, lds, tid)[0] * inv;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < K; k++)
      for (int e = 0; e < VE; e++) {
        const int i = k * VE + e;
        x[i] -= mean;
        s += e >= skip[k] ? x[i] * x[i] : 0.f;
      }
    const float rstd = 1.f / sqrtf(team_sum(f2{s, 0.f}, gl, lds, tid)[0] * inv + eps);
    char* to = a.y + (o * a.heads + head) * C * (i64)ESZ;
#if BACKWARD
    f2 m = {0.f, 0.f};
    for (int i = 0; i < K * VE; i++) {
      x[i] *= rstd;
      dw[i] += d[i] * x[i];
      db[i] += d[i];
      d[i] *= w[i];
      const bool in = i % VE >= skip[i / VE];
      m[0] += in ? d[i] : 0.f;
      m[1] += in ? d[i] * x[i] : 0.f;
    }
    m = team_sum(m, gl, lds, tid) * inv;
    for (int i = 0; i < K * VE; i++) x[i] = rstd * (d[i] - m[0] - x[i] * m[1]);
#else
    for (int i = 0; i < K * VE; i++) x[i] = x[i] * rstd * w[i] + b[i];
#endif
#pragma unroll
    for (int k = 0; k < K; k++) store_piece(to, start[k], skip[k], vec, x + k * VE);
  }
#if BACKWARD
  if (live)
    for (int k = 0; k < K; k++)
      for (int e = 0; e < VE; e++) {
        const int n = start[k] + e;
        if (e >= skip[k]) {
          if (a.dw) a.dw[team * C + n] = dw[k * VE + e];
          if (a.db) a.db[team * C + n] = db[k * VE + e];
        }
      }
#endif
}
