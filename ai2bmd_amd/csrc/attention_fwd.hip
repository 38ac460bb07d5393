// Fragment attention, forward: one pass over the keys with a running maximum and sum (attention.h has the tile).
//
// S^T = K Q^T puts keys in rows and queries in lanes; the softmax of a query is then 16 registers and one exchange with
// the other half of the wave, and O^T += V^T P^T takes P from the same registers.  16-bit rows take P in two parts (split8);
// maximum, sum and output stay in float32.
// Bound by vector instructions: 17 882 atoms, 8 heads of 32, bf16, with distances 1.62 ms (202 TFLOP/s of the two products; 347
// instructions per tile by the counters, the vector units busy throughout, the matrix units 13 %); 6007 atoms, 8 heads of 64,
// f16, with a table 0.24 ms (313 TFLOP/s; vector units busy 76 %) and 35 us of joining.
#include "attention.h"
#include "attention_host.h"

namespace vsn {

template <typename T, int DP, bool COOP>
__global__ __launch_bounds__(256, (forward_waves<T, DP>())) void k_attn_fwd(AttnParams p, size_t lds_per_wave) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lane_of_wave = lane;
  const int col = lane & 31, hi = lane >> 5;
  const int tid = COOP ? threadIdx.x : lane;
  constexpr int THREADS = COOP ? 64 * kCoopWaves : 64;
  const uint32_t id = COOP ? blockIdx.x : blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (uint32_t)p.count * p.heads) return;
  const int head = uniform(id % p.heads);
  const AttnWork w = load_work(p.work, uniform(id / p.heads));
  const AttnLds<T, DP> lds(lds_raw + (COOP ? 0 : wave * lds_per_wave));

  const int mine = (COOP ? wave * kTile : 0) + col;
  const bool live = mine < w.cols;
  const bool busy = (COOP ? wave * kTile : 0) < w.cols;  // wave-uniform
  const bool whole = (COOP ? wave * kTile : 0) + kTile <= w.cols;
  const int64_t row = (int64_t)w.col0 + (live ? mine : 0);
  const int kv = uniform(head / (p.heads / p.kv_heads));
  const T* kp = (const T*)p.k + kv * p.k_head;
  const T* vp = (const T*)p.v + kv * p.v_head;

  typename vec8<T>::type qf[DP / 16];
  const T* qp = (const T*)p.q + row * p.q_row + head * p.q_head;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) qf[c] = load_col<T>(qp, c * 16 + hi * 8, p.dim, live);
  const float scale = p.scale * kLog2e;
  float px = 0, py = 0, pz = 0, slope = 0;
  if (p.slope) {
    slope = p.slope[head] * kLog2e;
    px = p.q_pos[3 * row], py = p.q_pos[3 * row + 1], pz = p.q_pos[3 * row + 2];
  }
  int res = 0, res_lo = 0, res_hi = 0;
  if (p.table) {
    res = p.q_res[row];
    column_range(res, res_lo, res_hi);
    expand_table(lds.tab, p.table + (int64_t)head * p.n_buckets, p.lut, p.n_rel, tid, THREADS);
  }

  f32x16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) o[d] = acc_zero();
  float m = -INFINITY;  // the reference of the exponentials: that of the largest score so far
  LongSum l;            // this half's share

  TilePair<T, DP, THREADS> tiles;
  constexpr bool AHEAD = TilePair<T, DP, THREADS>::N <= 8;
  if (AHEAD && w.row0 < w.row1)
    tiles.load(kp + w.row0 * p.k_row, p.k_row, vp + w.row0 * p.v_row, p.v_row, w.row1 - w.row0, p.dim, tid);
  for (int k0 = w.row0; k0 < w.row1; k0 += kTile) {
    const int n = w.row1 - k0 < kTile ? w.row1 - k0 : kTile;
    if (!AHEAD) tiles.load(kp + k0 * p.k_row, p.k_row, vp + k0 * p.v_row, p.v_row, n, p.dim, tid);
    tile_sync<COOP>();
    tiles.store(lds.a, lds.b, n, p.dim, tid);
    if (tid < kTile) {
      const int64_t kr = k0 + (tid < n ? tid : 0);
      if (p.slope) lds.pos[tid] = make_float4(p.k_pos[3 * kr], p.k_pos[3 * kr + 1], p.k_pos[3 * kr + 2], 0.f);
      if (p.table) lds.res[tid] = p.k_res[kr];
    }
    tile_sync<COOP>();
    const int next = k0 + kTile;
    if (AHEAD && next < w.row1)
      tiles.load(kp + next * p.k_row, p.k_row, vp + next * p.v_row, p.v_row, w.row1 - next, p.dim, tid);
    if (!busy) continue;

    const int lane = here(lane_of_wave), col = lane & 31, hi = lane >> 5;
    f32x16 acc = acc_zero();
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
      if (c * 16 < p.dim) acc = Mma<T>::run(load_n<T, DP>(lds.a, c, col, hi), qf[c], acc);
    float s[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = acc[r] * scale;
    if (p.slope) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float4 k = lds.pos[acc_row(r, hi)];
        s[r] -= slope * pair_dist(px - k.x, py - k.y, pz - k.z);
      }
    }
    if (p.table) {
      const int end = clipped_end(lds.res[col], res_lo, res_hi, 1, p.reach);
      if (end >= 0) {  // far along the chain: one entry for the whole tile
        const float t = lds.tab[end];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] += t;
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] += lds.tab[rel_index(lds.res[acc_row(r, hi)], res, p.reach)];
      }
    }
    if (n < kTile || !whole) {
      const int limit = live ? n : 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = acc_row(r, hi) < limit ? s[r] : -INFINITY;
    }
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = fmaxf(m, exp_ref<T>(fmaxf(top, other_half(top))));
    // a row whose scores are all -inf so far keeps the maximum -inf and adds nothing
    const float ref = top == -INFINITY ? 0.f : top;
    const float fade = __builtin_amdgcn_exp2f(m - ref);
    m = top;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - ref);
    l.scale(fade);
    l.add(tile_sum(s));
    if (__any(fade != 1.f)) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= fade;
    }
    const Weights<T> p0 = split8<T>(s), p1 = split8<T>(s + 8);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      if (d * 32 >= p.dim) continue;
      tile_mma<T>(o[d], load_t<T, DP>(lds.b, 0, d * 32, lane, hi), p0, load_t<T, DP>(lds.b, 1, d * 32, lane, hi), p1);
    }
  }

  const float total = l.both_halves();
  if (!live) return;
  if (w.slot >= 0) {
    const int64_t at = ((int64_t)(w.slot + (COOP ? wave : 0)) * p.heads + head) * kTile + col;
    if (hi == 0) p.part_ml[at] = make_float2(m, total);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int e = d * 32 + 8 * g + 4 * hi;
        if (e < p.dim) store4<float>(p.part_o + at * p.dim + e, o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
      }
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (hi == 0 && p.stats) p.stats[head * p.rows_q + row] = attn_stats<T>(m, total);
  T* op = (T*)p.out + row * p.out_row + head * p.out_head;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int e = d * 32 + 8 * g + 4 * hi;
      if (e >= p.dim) continue;
      store4<T>(op + e, o[d][4 * g] * inv, o[d][4 * g + 1] * inv, o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv);
    }
}

// Joins the pieces' outputs, each weighted by 2^(m_s - max m), m the references of their exponentials.  A few pieces: one
// workgroup per (block of columns, head), a thread per four elements of a column, which finds the weights itself.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(AttnParams p) {
  const AttnJoin j = p.join[blockIdx.x];
  const int head = blockIdx.y, quads = p.dim / 4;
  for (int i = threadIdx.x; i < j.cols * quads; i += 256) {
    const int col = i / quads, d = i % quads * 4;
    const int64_t first = ((int64_t)j.slot0 * p.heads + head) * kTile + col, step = (int64_t)j.step * p.heads * kTile;
    float m = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < j.slots; ++s) m = fmaxf(m, p.part_ml[first + s * step].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < j.slots; ++s) {
      const float2 ml = p.part_ml[first + s * step];
      const float4 o = *(const float4*)(p.part_o + (first + s * step) * p.dim + d);
      const float f = __builtin_amdgcn_exp2f(ml.x - ref);
      l += f * ml.y;
      a.x += f * o.x, a.y += f * o.y, a.z += f * o.z, a.w += f * o.w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t row = (int64_t)j.col0 + col;
    store4<T>((T*)p.out + row * p.out_row + head * p.out_head + d, a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    if (d == 0 && p.stats) p.stats[head * p.rows_q + row] = attn_stats<T>(m, l);
  }
}

// Many pieces: one workgroup per (column, head).  The weights are put in LDS first, then dim / 4 lanes x (256 / (dim / 4))
// groups of pieces add up the rows.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join_many(AttnParams p) {
  __shared__ float weight[kMaxSlots];
  __shared__ float red[8];
  __shared__ float4 sum[256];
  const AttnJoin j = p.join[blockIdx.x / kTile];
  const int col = blockIdx.x % kTile, head = blockIdx.y, tid = threadIdx.x;
  if (col >= j.cols) return;
  const int64_t first = ((int64_t)j.slot0 * p.heads + head) * kTile + col, step = (int64_t)j.step * p.heads * kTile;
  float m = -INFINITY;
  for (int s = tid; s < j.slots; s += 256) m = fmaxf(m, p.part_ml[first + s * step].x);
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float ref = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int s = tid; s < j.slots; s += 256) {
    const float2 ml = p.part_ml[first + s * step];
    weight[s] = __builtin_amdgcn_exp2f(ml.x - ref);
    l += weight[s] * ml.y;
  }
  l = wave_sum(l);
  if ((tid & 63) == 0) red[4 + (tid >> 6)] = l;
  __syncthreads();
  l = red[4] + red[5] + red[6] + red[7];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t row = (int64_t)j.col0 + col;
  const int lanes = p.dim / 4, groups = 256 / lanes, g = tid / lanes, d = tid % lanes * 4;
  float4 a = make_float4(0, 0, 0, 0);
  if (g < groups)
    for (int s = g; s < j.slots; s += groups) {
      const float4 o = *(const float4*)(p.part_o + (first + s * step) * p.dim + d);
      const float f = weight[s];
      a.x += f * o.x, a.y += f * o.y, a.z += f * o.z, a.w += f * o.w;
    }
  sum[tid] = a;
  __syncthreads();
  if (g == 0) {
    for (int k = 1; k < groups; ++k) {
      const float4 o = sum[k * lanes + tid];
      a.x += o.x, a.y += o.y, a.z += o.z, a.w += o.w;
    }
    store4<T>((T*)p.out + row * p.out_row + head * p.out_head + d, a.x * inv, a.y * inv, a.z * inv, a.w * inv);
  }
  if (tid == 0 && p.stats) p.stats[head * p.rows_q + row] = attn_stats<T>(m, l);
}

template <typename T, int DP>
static int fwd_launch(const AttnPlanView& plan, AttnParams p, hipStream_t st) {
  const size_t bytes = AttnLds<T, DP>::bytes(p.table ? p.n_rel : 0);
  if (plan.lone) {
    p.work = plan.lone_work, p.count = plan.lone;
    const int64_t total = (int64_t)plan.lone * p.heads;
    const int waves = lone_waves(bytes);
    if (!allow_lds((const void*)k_attn_fwd<T, DP, false>, waves * bytes)) return -5;
    hipLaunchKernelGGL((k_attn_fwd<T, DP, false>), dim3((unsigned)((total + waves - 1) / waves)), dim3(64 * waves),
                       waves * bytes, st, p, bytes);
  }
  if (plan.coop) {
    p.work = plan.coop_work, p.count = plan.coop;
    if (!allow_lds((const void*)k_attn_fwd<T, DP, true>, bytes)) return -5;
    hipLaunchKernelGGL((k_attn_fwd<T, DP, true>), dim3((unsigned)((int64_t)plan.coop * p.heads)),
                       dim3(64 * kCoopWaves), bytes, st, p, bytes);
  }
  if (plan.few) {
    p.join = plan.join;
    hipLaunchKernelGGL((k_attn_join<T>), dim3(plan.few, p.heads), dim3(256), 0, st, p);
  }
  if (plan.joins > plan.few) {
    p.join = plan.join + plan.few;
    hipLaunchKernelGGL((k_attn_join_many<T>), dim3((plan.joins - plan.few) * kTile, p.heads), dim3(256), 0, st, p);
  }
  return hipGetLastError() == hipSuccess ? 0 : -5;
}

template <typename T>
static int fwd_dim(const AttnPlanView& plan, const AttnParams& p, hipStream_t st) {
  if (p.dim <= 32) return fwd_launch<T, 32>(plan, p, st);
  if (p.dim <= 64) return fwd_launch<T, 64>(plan, p, st);
  return fwd_launch<T, 128>(plan, p, st);
}

int attn_forward(int dtype, const AttnPlanView& plan, const AttnParams& p, hipStream_t st) {
  if (plan.small) {
    AttnParams small = p;
    small.work = plan.small_work, small.count = plan.small;
    const int rc = attn_small(dtype, small, small_groups(plan.small, p.kv_heads), false, st);
    if (rc) return rc;
  }
  switch (dtype) {
    case VSN_F32: return fwd_dim<float>(plan, p, st);
    case VSN_BF16: return fwd_dim<__bf16>(plan, p, st);
    default: return fwd_dim<_Float16>(plan, p, st);
  }
}

}  // namespace vsn
