// gfx950 kernel of rotary positions (include/mtc_serve.h).
//
// Pair i of a token at position p turns by p f_i. The angle is kept in turns, as a 64-bit fraction: p times
// round(2^64 f_i / 2 pi), modulo 2^64, is exact whatever the position, so far positions lose nothing and no table of
// cosines has to be kept (or read). The upper 32 bits are cut into a quadrant and an angle within an eighth of a turn either
// way, where sine and cosine are their Taylor series to x^9 and x^10 (the first terms left out: 1.8e-9 and 1e-10).

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <cmath>

#include "mtc_host.h"
#include "mtc_values.h"

#define MTC_API extern "C" __attribute__((visibility("default")))

using mtc::host::check_launch;
using mtc::host::fail;
using mtc::host::ok;
using namespace mtc::attn;

namespace {

constexpr int kRotaryThreads = 256;

__device__ __forceinline__ void sin_cos(int32_t position, uint64_t turns, float& s, float& c) {
  const uint64_t turn = (uint64_t)(int64_t)position * turns + 0x80000000u;
  const uint32_t t = (uint32_t)(turn >> 32), quadrant = (t + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(t - (quadrant << 30)) * 1.4629180792671596e-9f;      // 2 pi / 2^32
  const float z = x * x;
  float ps = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);                          // 1/9!, -1/7!
  ps = __builtin_fmaf(z, ps, 8.3333333e-3f);
  ps = __builtin_fmaf(z, ps, -1.6666667e-1f);
  const float sx = __builtin_fmaf(x * z, ps, x);
  float pc = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);                          // -1/10!, 1/8!
  pc = __builtin_fmaf(z, pc, -1.3888889e-3f);
  pc = __builtin_fmaf(z, pc, 4.1666667e-2f);
  pc = __builtin_fmaf(z, pc, -0.5f);
  const float cx = __builtin_fmaf(z, pc, 1.0f);
  const bool odd = quadrant & 1;
  const float a = odd ? cx : sx, b = odd ? sx : cx;
  s = quadrant & 2 ? -a : a;
  c = (quadrant + 1) & 2 ? -b : b;
}

// One thread per VEC pairs of a token, for HEADS heads: their sines and cosines serve all of them. Slots past the
// turned dims copy 2 VEC elements each.
// Bound by memory where there are many tokens (16384 of 32 + 8 heads of 128 bf16: 336 MB in 69 us, 4.9 TB/s; a 1 GiB copy: 5.14), by the
// launch where there are few (one token 2.6 to 3.1 us).
template <int DT, int VEC, int HEADS>
__global__ __launch_bounds__(kRotaryThreads) void k_rotary(const mtc_rotary_args a) {
  using V = Value<DT>;
  typedef typename V::type T;
  typedef Run<T, VEC> R;
  const int slots = a.dim / (2 * VEC), pairs = a.rotated / (2 * VEC), all = a.heads + a.kv_heads;
  const int groups = (all + HEADS - 1) / HEADS;
  const int64_t i = (int64_t)blockIdx.x * kRotaryThreads + threadIdx.x;
  const int slot = (int)(i % slots);
  const int64_t rest = i / slots;
  const int h0 = (int)(rest % groups) * HEADS;
  const int64_t row = rest / groups;
  if (row >= a.rows) return;
  const bool turn = slot < pairs;
  int first, second;                       // elements of the slot's two runs
  if (!turn || a.interleaved) {
    first = slot * 2 * VEC;
    second = first + VEC;
  } else {
    first = slot * VEC;
    second = a.rotated / 2 + first;
  }
  R x[HEADS], y[HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = h0 + j;
    if (h >= all) break;
    const mtc_heads& in = h < a.heads ? a.q : a.k;
    const T* p = reinterpret_cast<const T*>(in.data) + row * in.row_stride + (int64_t)(h < a.heads ? h : h - a.heads) * in.head_stride;
    x[j] = *reinterpret_cast<const R*>(p + first);
    y[j] = *reinterpret_cast<const R*>(p + second);
  }
  float s[VEC], c[VEC];
  if (turn) {
    const int32_t position = a.positions[row];
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      sin_cos(position, a.turns[slot * VEC + k], s[k], c[k]);
      s[k] *= a.amplitude;
      c[k] *= a.amplitude;
    }
  }
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = h0 + j;
    if (h >= all) break;
    if (turn) {
      if (a.interleaved) {
        T z[2 * VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          z[k] = x[j].x[k];
          z[VEC + k] = y[j].x[k];
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float u = V::get(z[2 * k]), v = V::get(z[2 * k + 1]);
          z[2 * k] = V::put(__builtin_fmaf(u, c[k], -(v * s[k])));
          z[2 * k + 1] = V::put(__builtin_fmaf(u, s[k], v * c[k]));
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          x[j].x[k] = z[k];
          y[j].x[k] = z[VEC + k];
        }
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float u = V::get(x[j].x[k]), v = V::get(y[j].x[k]);
          x[j].x[k] = V::put(__builtin_fmaf(u, c[k], -(v * s[k])));
          y[j].x[k] = V::put(__builtin_fmaf(u, s[k], v * c[k]));
        }
      }
    }
    const mtc_heads& to = h < a.heads ? a.oq : a.ok;
    T* p = reinterpret_cast<T*>(to.data) + row * to.row_stride + (int64_t)(h < a.heads ? h : h - a.heads) * to.head_stride;
    *reinterpret_cast<R*>(p + first) = x[j];
    *reinterpret_cast<R*>(p + second) = y[j];
  }
}

int check_rotary_heads(const char* what, const mtc_heads& x, int align) {
  if (!x.data) return fail(MTC_E_NULL, "%s is NULL", what);
  if ((uintptr_t)x.data % 16) return fail(MTC_E_SHAPE, "%s must be 16-byte aligned", what);
  if (x.row_stride < 0 || x.head_stride < 0 || x.row_stride % align || x.head_stride % align)
    return fail(MTC_E_SHAPE, "%s: strides %lld, %lld must be non-negative multiples of %d elements", what, (long long)x.row_stride,
                (long long)x.head_stride, align);
  return MTC_OK;
}

template <int DT, int VEC>
int launch_rotary(const mtc_rotary_args& a, hipStream_t st) {
  const int64_t units = (int64_t)a.rows * (a.dim / (2 * VEC)), all = a.heads + a.kv_heads;
  // sines for four heads at once where that still fills the chip, 512 threads a CU. Measured in a graph, one head and four a thread, by the
  // count of threads of four (K): 32 + 8 heads of 128, 512 tokens (40) 4.5, 5.3 us; 1228 (96) 6.8, 7.1; 1400 (109) 7.4, 7.6; 1500 (117) 8.2, 7.8; 1638
  // (128) 8.3, 8.2; 2048 (160) 10.8, 9.5; 4096 17.0, 15.1; 14 + 2 of 64, 6000 (94) 6.7, 7.3; 8192 (128) 8.4, 8.1; 8 + 1 of 128, 6144 (144) 7.7, 8.6;
  // 8192 (192) 9.9, 9.1; 16 + 16 of 80, 32 turned, 3200 (125) 8.3, 9.1. fp32 would cross later: 32 + 8 of 128, 2048 (160) 16.0, 17.5.
  constexpr int kHeads = 4;
  const bool few = units * ((all + kHeads - 1) / kHeads) < 128 * 1024;
  const int64_t threads = units * (few ? all : (all + kHeads - 1) / kHeads);
  const int64_t blocks = (threads + kRotaryThreads - 1) / kRotaryThreads;
  if (blocks > 0xFFFFFF) return fail(MTC_E_SHAPE, "%d rows of %d heads: too many", a.rows, (int)all);
  if (few) k_rotary<DT, VEC, 1><<<(unsigned)blocks, kRotaryThreads, 0, st>>>(a);
  else k_rotary<DT, VEC, kHeads><<<(unsigned)blocks, kRotaryThreads, 0, st>>>(a);
  return check_launch("k_rotary");
}
// Runs of the largest power of two that divides half of the turned and half of the other dims.
template <int DT>
int launch_rotary(const mtc_rotary_args& a, hipStream_t st) {
  const int both = a.rotated | a.dim;
  if (both % 16 == 0) return launch_rotary<DT, 8>(a, st);
  if (both % 8 == 0) return launch_rotary<DT, 4>(a, st);
  if (both % 4 == 0) return launch_rotary<DT, 2>(a, st);
  return launch_rotary<DT, 1>(a, st);
}

}  // namespace

MTC_API int mtc_rotary(const mtc_rotary_args* a, void* hip_stream) {
  if (!a) return fail(MTC_E_NULL, "args is NULL");
  if (a->abi_version != MTC_ABI_VERSION) return fail(MTC_E_VERSION, "args of ABI %u, library %d", a->abi_version, MTC_ABI_VERSION);
  if (a->dtype != MTC_DTYPE_F32 && a->dtype != MTC_DTYPE_BF16 && a->dtype != MTC_DTYPE_F16)
    return fail(MTC_E_DTYPE, "rotary positions take fp32, bf16 or f16, got dtype %d", a->dtype);
  if (a->rows < 0 || a->heads < 0 || a->kv_heads < 0 || a->heads > 0xFFFF || a->kv_heads > 0xFFFF)
    return fail(MTC_E_SHAPE, "%d rows of %d and %d heads", a->rows, a->heads, a->kv_heads);
  if (a->dim < 8 || a->dim > MTC_ROTARY_MAX_DIM || a->dim % 8)
    return fail(MTC_E_SHAPE, "head size %d: a multiple of 8 from 8 to %d", a->dim, MTC_ROTARY_MAX_DIM);
  if (a->reserved != 0) return fail(MTC_E_SHAPE, "reserved must be 0");
  if (a->rotated < 2 || a->rotated > a->dim || a->rotated % 2) return fail(MTC_E_SHAPE, "%d of %d dims turned: an even count", a->rotated, a->dim);
  if (!std::isfinite(a->amplitude)) return fail(MTC_E_SHAPE, "amplitude must be finite");
  if (a->rows == 0 || a->heads + a->kv_heads == 0) return ok();
  if (!a->positions || !a->turns) return fail(MTC_E_NULL, "positions or turns is NULL");
  const int align = a->dtype == MTC_DTYPE_F32 ? 4 : 8;
  if (a->heads) {
    if (int rc = check_rotary_heads("q", a->q, align)) return rc;
    if (int rc = check_rotary_heads("oq", a->oq, align)) return rc;
  }
  if (a->kv_heads) {
    if (int rc = check_rotary_heads("k", a->k, align)) return rc;
    if (int rc = check_rotary_heads("ok", a->ok, align)) return rc;
  }
  hipStream_t st = (hipStream_t)hip_stream;
  if (a->dtype == MTC_DTYPE_F32) return launch_rotary<MTC_DTYPE_F32>(*a, st);
  if (a->dtype == MTC_DTYPE_BF16) return launch_rotary<MTC_DTYPE_BF16>(*a, st);
  return launch_rotary<MTC_DTYPE_F16>(*a, st);
}
