// out[x] = sum over s of in[s][x]: fp32 summed in 64 bits and rounded once, in a fixed order.  Used for gradients of what
// several workgroups share: heads that share keys (few slices, many columns), norm weights, a decay that all tokens share
// (many slices, few columns).  A workgroup takes `cw` columns and deals the slices to its 256 / cw rows of threads; with
// more than one part each part sums a range of slices into its own row of `out` (fp32), and a second launch joins them.
// Bound by memory where there is much (2 slices of 4 M columns: 12 us, 50 MB), else by the launch: 512 slices of 4096 columns, twice,
// 5 us, and 4 us for the second launch.
#include <hip/hip_runtime.h>

typedef long long i64;
typedef float f4 __attribute__((ext_vector_type(4)));

struct Args {
  struct {
    const float* in;
    char* out;
  } pair[2];                       // blockIdx.y chooses
  i64 S, X, type, cw, parts;       // type: 0 bfloat16, 1 float16, 2 float32; cw: a power of two from 1 to 256, or 1024: see below
};

static __device__ __forceinline__ void store(char* out, i64 at, int type, float v) {
  if (type == 2) ((float*)out)[at] = v;
  else if (type == 1) ((_Float16*)out)[at] = (_Float16)v;
  else ((__bf16*)out)[at] = (__bf16)v;
}

extern "C" __global__ void __launch_bounds__(256) slice_sum(Args a) {
  __shared__ double part[256];
  const float* in = a.pair[blockIdx.y].in;
  char* out = a.pair[blockIdx.y].out;
  if (a.cw > 256) {                // few slices: a thread sums all of them, four neighbouring columns at a time
    const i64 x = ((i64)blockIdx.x * 256 + threadIdx.x) * 4;
    if (x >= a.X) return;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
    for (i64 i = 0; i < a.S; i++) {
      const f4 v = *(const f4*)(in + i * a.X + x);
      for (int c = 0; c < 4; c++) s[c] += (double)v[c];
    }
    for (int c = 0; c < 4; c++) store(out, x + c, (int)a.type, (float)s[c]);
    return;
  }
  const int tid = threadIdx.x, cw = (int)a.cw, col = tid % cw, row = tid / cw, nr = 256 / cw;
  const i64 groups = (a.X + cw - 1) / cw, x = (i64)(blockIdx.x % groups) * cw + col, pt = blockIdx.x / groups;
  const i64 per = (a.S + a.parts - 1) / a.parts, s0 = pt * per, s1 = s0 + per < a.S ? s0 + per : a.S;
  double s = 0.0;
  if (x < a.X) {
    i64 i = s0 + row;
    for (; i + 3 * nr < s1; i += 4 * nr) {
      const float v0 = in[i * a.X + x], v1 = in[(i + nr) * a.X + x], v2 = in[(i + 2 * nr) * a.X + x], v3 = in[(i + 3 * nr) * a.X + x];
      s += (double)v0 + (double)v1 + ((double)v2 + (double)v3);
    }
    for (; i < s1; i += nr) s += (double)in[i * a.X + x];
  }
  part[tid] = s;
  __syncthreads();
  for (int n = nr / 2; n > 0; n /= 2) {
    if (row < n) part[tid] += part[tid + n * cw];
    __syncthreads();
  }
  if (row == 0 && x < a.X) store(out, pt * a.X + x, (int)a.type, (float)part[col]);
}
