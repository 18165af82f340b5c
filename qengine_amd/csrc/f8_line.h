// f8_line.h -- work of ragged batches as one line of units that is cut into equal parts, shared by
// attn_f8.hip and weigh_f8.hip.
#pragma once
#include <hip/hip_runtime.h>

namespace qkv {

namespace {

// Inclusive sums over the lanes, none above `top`
__device__ __forceinline__ int scan64(int v, int top) {
  auto add = [&](int o) { v = min(v + o, top); };
  add(__builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));   // within rows of 16, from 1, 2, 4, 8 lanes below
  add(__builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));   // the row before, the half before
  add(__builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return v;
}

// Sums stop at kLineMax: starts that are not in order can name the same rows many times, and the
// line of them all may pass 32 bits.
constexpr int kLineMax = (1 << 30) - 1;
__device__ __forceinline__ int add_units(int a, int b) { return min(a + b, kLineMax); }

template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int* lds, int& sum) {   // inclusive
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  v = scan64(v, kLineMax);
  __syncthreads();
  if (lane == 63) lds[w] = v;
  __syncthreads();
  int before = 0;
  sum = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) {
    if (i < w) before = add_units(before, lds[i]);
    sum = add_units(sum, lds[i]);
  }
  return add_units(v, before);
}

// Parts of the line: at most a workgroup's each and none empty, the first `more` of them one
// unit longer (the units of all heads stay below 2^31: the host sees to it).
struct Parts {
  int n, q, more;
  __device__ __forceinline__ Parts(int units, int groups) {
    n = min(units, groups);
    q = n > 0 ? units / n : 0;
    more = units - q * n;
  }
  __device__ __forceinline__ int begin(int g) const { return g * q + min(g, more); }
  __device__ __forceinline__ int of(int x) const {   // the part that holds unit x
    const int lo = more * (q + 1);
    return x < lo ? x / (q + 1) : more + (x - lo) / q;
  }
};

}  // namespace

}  // namespace qkv
