// Layer norm over the last axis, forward and backward with the gradients of weight and bias, as an operator of its own
// (the ViS-MP layer's torch.nn.LayerNorm, ViSNet/model/visnet_block.py:180,237; the engine's node walks hold the same
// norm fused and need only its input adjoint).
//
//   h = (x - mean) rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = h w + b
//   g = dy w,  dx = rstd (g - mean(g) - h mean(g h)),  dw = sum_rows dy h,  db = sum_rows dy
//
// Bound by memory: x and y once forward; x, dy and dx once backward.  LPR lanes hold one row in registers (NV vectors of
// 16 bytes each), so the mean is subtracted before the squares are summed and nothing is read twice; narrow rows put
// 64 / LPR rows into a wave.  A lane keeps its columns for all the rows it visits: weight and bias stay in registers, and
// so do the column sums of the backward pass, which are joined over the workgroup in LDS and over the workgroups by a
// second launch, both in a fixed order (no atomics: equal inputs give equal bits).  All sums are float32.
// Vector loads need only element alignment (gfx950 takes global addresses of any alignment); the row's last, partial
// vector is stored element by element.
// One MI355X (a large copy runs at 4.73 TB/s): forward 1 310 720 x 256 f32 0.45 ms (5.9 TB/s); 80 000 x 256 bf16 forward 16 us
// (5.2, from the cache), backward 24 us (5.1) and 4 us for the second launch; 30 011 x 509 f16, rows at any address, 15 and
// 21 us (4.1, 4.4) and 4 us.
#include "typed.h"

namespace vsn {

// Columns at ... at + VEC of a row, zeros behind its end.  ODD (16-bit rows of at least one vector that end within one): a lane
// at the row's end loads the row's last whole vector and shifts its columns down, as nobody waits then for one that goes
// element by element (30 011 x 509 f16: forward 17.5 -> 14.5 us, both directions 52.9 -> 37.1).  Rows of whole vectors keep the
// branch: 80 000 rows bf16 forward, width 256 15.6 us and 16.5 this way, 192 13.4 and 14.2, 320 21.2 and 22.3; only the
// backward pass gains at 320 (both directions 58.0 and 54.4).  So do float32 rows: 1 310 720 x 256 forward 454 us, 634 this way.
template <typename T, int VEC, bool ODD>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int at, int width, float (&v)[VEC]) {
  if constexpr (ODD) {
    static_assert(sizeof(T) * VEC == 16, "one 16-byte vector");
    const int from = __builtin_elementwise_min(at, width - VEC), skip = at - from;
    unsigned __int128 bits;
    __builtin_memcpy(&bits, p + from, sizeof(bits));
    if (skip) bits = skip < VEC ? bits >> (skip * (int)sizeof(T) * 8) : 0;
    T tmp[VEC];
    __builtin_memcpy(tmp, &bits, sizeof(tmp));
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (float)tmp[i];
  } else if (at + VEC <= width) {
    T tmp[VEC];
    __builtin_memcpy(tmp, p + at, sizeof(tmp));
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = (float)tmp[i];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = at + i < width ? (float)p[at + i] : 0.f;
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_row(T* __restrict__ p, int at, int width, const float (&v)[VEC]) {
  if (at + VEC <= width) {
    T tmp[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) tmp[i] = (T)v[i];
    __builtin_memcpy(p + at, tmp, sizeof(tmp));
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (at + i < width) p[at + i] = (T)v[i];
  }
}
// weight / bias columns of one lane: the rows' type or float32; absent = `fill`.  Whole vectors, as the rows are: a load per
// element made up almost half of the forward pass (80 000 x 256 bf16 27 us, so 15 us; 5000 x 1024 bf16 13.4 us, so 6.0 us).
template <typename T, int VEC, bool ODD>
__device__ __forceinline__ void load_param(const void* p, int is_f32, int at, int width, float fill, float (&v)[VEC]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = at + i < width ? fill : 0.f;
  } else if (is_f32) {
    load_row<float, VEC, false>((const float*)p, at, width, v);
  } else {
    load_row<T, VEC, ODD>((const T*)p, at, width, v);
  }
}
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// (y may be x: a wave holds its rows before it stores them, and no other wave reads them)
template <typename T, int VEC, int LPR, int NV, bool ODD>
__global__ __launch_bounds__(256) void k_layernorm(const T* x, int64_t ldx, const void* __restrict__ w,
                                                   const void* __restrict__ b, int param_f32, int64_t rows, int width,
                                                   float inv_width, float eps, T* y, int64_t ldy,
                                                   float2* __restrict__ stats) {
  constexpr int RPB = 256 / LPR;  // rows of a workgroup per turn
  const int lane = threadIdx.x % LPR;
  float wv[NV][VEC], bv[NV][VEC];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    load_param<T, VEC, ODD>(w, param_f32, (n * LPR + lane) * VEC, width, 1.f, wv[n]);
    load_param<T, VEC, ODD>(b, param_f32, (n * LPR + lane) * VEC, width, 0.f, bv[n]);
  }
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; row < rows; row += (int64_t)gridDim.x * RPB) {
    float v[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      load_row<T, VEC, ODD>(x + row * ldx, (n * LPR + lane) * VEC, width, v[n]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += v[n][i];
    }
    const float mean = row_sum<LPR>(s) * inv_width;
    float q = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[n][i] = (n * LPR + lane) * VEC + i < width ? v[n][i] - mean : 0.f;
        q += v[n][i] * v[n][i];
      }
    const float rstd = 1.f / sqrtf(row_sum<LPR>(q) * inv_width + eps);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[n][i] = v[n][i] * rstd * wv[n][i] + bv[n][i];
      store_row<T, VEC>(y + row * ldy, (n * LPR + lane) * VEC, width, v[n]);
    }
    if (stats && lane == 0) stats[row] = make_float2(mean, rstd);
  }
}

// partial: [gridDim.x][2][width] column sums of dy h and dy.  (dx may be dy, as y may be x above: no restrict on either.)
template <typename T, int VEC, int LPR, int NV, bool ODD>
__global__ __launch_bounds__(256) void k_layernorm_bwd(const T* dy, int64_t lddy, const T* __restrict__ x,
                                                       int64_t ldx, const float2* __restrict__ stats,
                                                       const void* __restrict__ w, int param_f32, int64_t rows,
                                                       int width, float inv_width, T* dx, int64_t lddx,
                                                       float* __restrict__ partial) {
  constexpr int RPB = 256 / LPR;
  const int lane = threadIdx.x % LPR;
  float wv[NV][VEC], aw[NV][VEC], ab[NV][VEC];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    load_param<T, VEC, ODD>(w, param_f32, (n * LPR + lane) * VEC, width, 1.f, wv[n]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) aw[n][i] = ab[n][i] = 0.f;
  }
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; row < rows; row += (int64_t)gridDim.x * RPB) {
    const float2 st = stats[row];
    float h[NV][VEC], g[NV][VEC];
    float sg = 0.f, sgh = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      load_row<T, VEC, ODD>(x + row * ldx, (n * LPR + lane) * VEC, width, h[n]);
      load_row<T, VEC, ODD>(dy + row * lddy, (n * LPR + lane) * VEC, width, g[n]);
    }
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[n][i] = (n * LPR + lane) * VEC + i < width ? (h[n][i] - st.x) * st.y : 0.f;
        aw[n][i] += g[n][i] * h[n][i];
        ab[n][i] += g[n][i];
        g[n][i] *= wv[n][i];
        sg += g[n][i];
        sgh += g[n][i] * h[n][i];
      }
    sg = row_sum<LPR>(sg) * inv_width;
    sgh = row_sum<LPR>(sgh) * inv_width;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) g[n][i] = st.y * (g[n][i] - sg - h[n][i] * sgh);
      store_row<T, VEC>(dx + row * lddx, (n * LPR + lane) * VEC, width, g[n]);
    }
  }
  if (!partial) return;
  // the RPB row groups of the workgroup hold the same columns: added one after the other, in their order
  __shared__ float sw[NV * LPR * VEC], sb[NV * LPR * VEC];
  for (int r = 0; r < RPB; ++r) {
    if ((int)threadIdx.x / LPR == r)
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int c = (n * VEC + i) * LPR + lane;  // lanes side by side: no bank is hit twice
          sw[c] = r ? sw[c] + aw[n][i] : aw[n][i];
          sb[c] = r ? sb[c] + ab[n][i] : ab[n][i];
        }
    __syncthreads();
  }
  float* out = partial + (size_t)blockIdx.x * 2 * width;
  for (int c = threadIdx.x; c < width; c += 256) {
    const int n = c / (LPR * VEC), l = c / VEC % LPR, i = c % VEC;
    out[c] = sw[(n * VEC + i) * LPR + l];
    out[width + c] = sb[(n * VEC + i) * LPR + l];
  }
}

// dw and db from the workgroups' partial sums: 16 columns x 64 strided rows of partials per workgroup, so that a lane's
// chain of loads is short (1024 partials: 16 loads; with 8 rows per workgroup 128 loads took 39 us of a 95 us pass)
template <typename T>
__global__ __launch_bounds__(1024) void k_layernorm_params(const float* __restrict__ partial, int groups, int width,
                                                          void* __restrict__ dw, void* __restrict__ db,
                                                          int param_f32) {
  __shared__ float red[64][17];
  const int c = blockIdx.x * 16 + threadIdx.x % 16, r = threadIdx.x / 16;
  const int which = blockIdx.y;
  float s = 0.f;
  if (c < width)
#pragma unroll 4
    for (int g = r; g < groups; g += 64) s += partial[((size_t)g * 2 + which) * width + c];
  red[r][threadIdx.x % 16] = s;
  __syncthreads();
  if (r < 8) {
#pragma unroll
    for (int k = 8; k < 64; k += 8) s += red[r + k][threadIdx.x % 16];
    red[r][threadIdx.x % 16] = s;
  }
  __syncthreads();
  void* out = which ? db : dw;
  if (r == 0 && c < width && out) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][threadIdx.x];
    if (param_f32)
      ((float*)out)[c] = s;
    else
      ((T*)out)[c] = (T)s;
  }
}

constexpr int kNormWidth = 4096;
constexpr int kNormGroups = 1024;

static int norm_groups(int64_t rows, int rows_per_group, int cap) {
  const int64_t need = (rows + rows_per_group - 1) / rows_per_group;
  return (int)(need < cap ? need : cap);
}

// Workgroups of the forward pass.  As many as the chip holds at once, each walking its share of the rows, so that weight and
// bias are read once for many rows: 80 000 x 256 bf16 15.6 us, with one turn each 18.9; 30 011 x 509 f16 13.8 and 16.7;
// 1 310 720 x 80 bf16 83 and 155; 700 000 x 509 f16 382 and 396; 150 000 x 4096 f32 973 and 1111.  Float32 rows of ordinary
// width that do not fit the 256 MB cache go the other way, as fresh waves keep more loads in flight than a wave's next turn:
// 1 310 720 x 256 f32 552 us walking, 449 with one turn each; 200 000 x 256 78 and 72; 2 600 000 x 64 274 and 222;
// 600 000 x 1024 984 and 853.  But not where lanes of a row's only vector lie behind its end, or half of the lanes have no
// second one: each load then waits for the one before (load_row), which a fresh wave pays for weight, bias and row alike.
// 96 10^6 elements f32, walking and one turn each: width 96 147 and 215 us, 192 145 and 217, 240 150 and 177, 288 156 and 183,
// 320 154 and 167, 352 155 and 155; 384 154 and 147, 448 151 and 136, 640 151 and 140; 64, 128 and 256 149 and 132.
template <typename T>
static int norm_forward_cap(int64_t rows, int width) {
  const bool beyond_cache = rows * width * 2 * (int64_t)sizeof(T) > (int64_t)256 << 20;
  const bool lanes_full = width <= 256 ? (width & (width - 1)) == 0 : width >= 384;
  return sizeof(T) == 4 && width >= 64 && width <= 1024 && lanes_full && beyond_cache ? 1 << 20 : 2048;
}

struct NormArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx, *dw, *db;
  float *stats, *partial;
  int64_t ldx, ldy, lddy, lddx, rows;
  int width, param_f32;
  float eps;
  bool backward;
};

template <typename T, int VEC, int LPR, int NV, bool ODD>
static void norm_launch(const NormArgs& a, hipStream_t st) {
  const float inv = 1.0f / (float)a.width;
  const int rpb = 256 / LPR;
  if (!a.backward) {
    if (!a.rows) return;
    const int groups = norm_groups(a.rows, rpb, norm_forward_cap<T>(a.rows, a.width));
    hipLaunchKernelGGL((k_layernorm<T, VEC, LPR, NV, ODD>), dim3(groups), dim3(256), 0, st,
                       (const T*)a.x, a.ldx, a.w, a.b, a.param_f32, a.rows, a.width, inv, a.eps, (T*)a.y, a.ldy,
                       (float2*)a.stats);
    return;
  }
  const int groups = norm_groups(a.rows, rpb, kNormGroups);
  float* partial = a.dw || a.db ? a.partial : nullptr;
  if (groups)
    hipLaunchKernelGGL((k_layernorm_bwd<T, VEC, LPR, NV, ODD>), dim3(groups), dim3(256), 0, st, (const T*)a.dy, a.lddy,
                       (const T*)a.x, a.ldx, (const float2*)a.stats, a.w, a.param_f32, a.rows, a.width, inv, (T*)a.dx,
                       a.lddx, partial);
  if (partial || (!groups && (a.dw || a.db)))
    hipLaunchKernelGGL((k_layernorm_params<T>), dim3((a.width + 15) / 16, 2), dim3(1024), 0, st, partial, groups,
                       a.width, a.dw, a.db, a.param_f32);
}

template <typename T, int VEC, bool ODD>
static void norm_pick(const NormArgs& a, hipStream_t st) {
  const int n = a.width;
  if (n <= 8 * VEC) return norm_launch<T, VEC, 8, 1, ODD>(a, st);
  if (n <= 16 * VEC) return norm_launch<T, VEC, 16, 1, ODD>(a, st);
  if (n <= 32 * VEC) return norm_launch<T, VEC, 32, 1, ODD>(a, st);
  if (n <= 64 * VEC) return norm_launch<T, VEC, 64, 1, ODD>(a, st);
  if (n <= 128 * VEC) return norm_launch<T, VEC, 64, 2, ODD>(a, st);
  if (n <= 256 * VEC) return norm_launch<T, VEC, 64, 4, ODD>(a, st);
  if (n <= 512 * VEC) return norm_launch<T, VEC, 64, 8, ODD>(a, st);
  if constexpr (VEC == 4) return norm_launch<T, VEC, 64, 16, ODD>(a, st);
}

template <typename T>
static void norm_pick_16bit(const NormArgs& a, hipStream_t st) {
  if (a.width % 8 && a.width > 8)
    norm_pick<T, 8, true>(a, st);
  else
    norm_pick<T, 8, false>(a, st);
}

static int norm_dispatch(int dtype, const NormArgs& a, hipStream_t st) {
  switch (dtype) {
    case VSN_F32: norm_pick<float, 4, false>(a, st); break;
    case VSN_BF16: norm_pick_16bit<__bf16>(a, st); break;
    default: norm_pick_16bit<_Float16>(a, st); break;
  }
  return hipGetLastError() == hipSuccess ? 0 : -5;
}

static bool norm_bad(int dtype, int param_dtype, int64_t rows, int width) {
  return dtype < VSN_F32 || dtype > VSN_F16 || (param_dtype != dtype && param_dtype != VSN_F32) || rows < 0 ||
         width < 1 || width > kNormWidth;
}

}  // namespace vsn

extern "C" int vsn_layernorm(int device_id, int dtype, int param_dtype, const void* dev_x, int64_t ldx,
                             const void* dev_w, const void* dev_b, int64_t rows, int width, float eps, void* dev_y,
                             int64_t ldy, float* dev_stats, void* stream) {
  if (vsn::norm_bad(dtype, param_dtype, rows, width) || !(eps >= 0.f)) return -22;
  if (rows && (!dev_x || !dev_y || ldx < width || ldy < width)) return -22;
  vsn::DeviceScope scope(device_id);
  if (!scope.ok) return -19;
  vsn::NormArgs a = {};
  a.x = dev_x, a.w = dev_w, a.b = dev_b, a.y = dev_y, a.stats = dev_stats;
  a.ldx = ldx, a.ldy = ldy, a.rows = rows, a.width = width, a.param_f32 = param_dtype == VSN_F32, a.eps = eps;
  return vsn::norm_dispatch(dtype, a, (hipStream_t)stream);
}

extern "C" int64_t vsn_layernorm_workspace(int64_t rows, int width) {
  if (rows < 0 || width < 1 || width > vsn::kNormWidth) return -22;
  // at least 4 rows per workgroup, whatever the lanes per row (norm_launch)
  const int64_t groups = rows / 4 + 1 < vsn::kNormGroups ? rows / 4 + 1 : vsn::kNormGroups;
  return groups * 2 * width * (int64_t)sizeof(float);
}

extern "C" int vsn_layernorm_backward(int device_id, int dtype, int param_dtype, const void* dev_dy, int64_t lddy,
                                      const void* dev_x, int64_t ldx, const float* dev_stats, const void* dev_w,
                                      int64_t rows, int width, void* dev_dx, int64_t lddx, void* dev_dw, void* dev_db,
                                      void* dev_workspace, int64_t workspace_bytes, void* stream) {
  if (vsn::norm_bad(dtype, param_dtype, rows, width)) return -22;
  if (rows && (!dev_dy || !dev_x || !dev_stats || !dev_dx || lddy < width || ldx < width || lddx < width)) return -22;
  if (rows && (dev_dw || dev_db) && (!dev_workspace || workspace_bytes < vsn_layernorm_workspace(rows, width)))
    return -22;
  vsn::DeviceScope scope(device_id);
  if (!scope.ok) return -19;
  vsn::NormArgs a = {};
  a.backward = true;
  a.dy = dev_dy, a.x = dev_x, a.w = dev_w, a.dx = dev_dx, a.dw = dev_dw, a.db = dev_db;
  a.stats = (float*)dev_stats, a.partial = (float*)dev_workspace;
  a.lddy = lddy, a.ldx = ldx, a.lddx = lddx, a.rows = rows, a.width = width, a.param_f32 = param_dtype == VSN_F32;
  return vsn::norm_dispatch(dtype, a, (hipStream_t)stream);
}
