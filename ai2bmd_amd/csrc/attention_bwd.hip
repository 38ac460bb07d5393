// Fragment attention, backward (attention.h has the tile; formulas of the forward pass there).
//
//   P = 2^(s - m) / l (s in units of log 2),  dP_ij = do_i.v_j,  D_i = sum_j P_ij dP_ij,  dS = P (dP - D)
//   dq_i = scale sum_j dS k_j      dk_j = scale sum_i dS q_i      dv_j = sum_i P do_i
//   dslope_a = - sum dS r          dtable[a][b] = sum over the pairs of bucket b
//   dx_i -= slope dS (x_i - x_j) / r,  dx_j -= the opposite; summed over heads
//
// Two passes that both recompute the scores, each with its sums in registers and nothing to add atomically: queries in
// lanes for dq, D, the slopes, the table and the queries' share of the positions; keys in lanes for dk, dv and the keys'
// share.  Seven products instead of five, against a pass that would have to add dq (or dk, dv) across workgroups in an
// order of its own.  The maximum and the sum are kept apart (not as one logarithm), so P keeps its precision however
// large the scores are.  D is summed from the scores before anything is rounded (do_i.o_i would carry the rounding of the
// output into every float32 gradient): a pass of its own ahead of the dq pass, except where one tile
// holds all keys of a fragment and everything is still in registers.
// Long runs of rows are split into pieces of equal length (make_lists); a piece leaves float32 sums that a join adds up.
// P and dS enter a product in two parts of 16-bit rows' type (split8).  float16 has few exponents for that: P goes in
// times 2^14, and dS times a power of two per column that follows the largest one seen so far.
// All sums are in a fixed order; the table's are kept per wave in LDS.
// 17 882 atoms, 8 heads of 32, bf16, distances and table: D 1.5 ms, dq 3.1 ms, dk / dv 3.7 ms, bound by vector instructions
// (the units busy 95, 91 and 85 % by the counters); 6007 atoms, 8 heads of 64, f16, table: 0.18, 0.60 and 0.48 ms (69, 39 and
// 54 %: the two waves per SIMD that registers allow wait for LDS and for one another).
#include "attention.h"
#include "attention_host.h"

namespace vsn {

// a column's power of two for float16 gradients: keeps max |dS| scale below 2^15
struct ColumnScale {
  float f = 0x1p100f;
  // the factor by which what was summed so far has to be multiplied, 1 where the scale stays
  __device__ __forceinline__ float follow(float largest) {
    if (largest * f <= 0x1p15f || !(largest < INFINITY)) return 1.f;
    const float next = ldexpf(1.f, 14 - ilogbf(largest));
    const float change = next / f;
    f = next;
    return change;
  }
};

// DELTA: the pass for D of fragments of several tiles; else the dq pass
template <typename T, int DP, bool COOP, bool DELTA>
__global__ __launch_bounds__(256, (backward_waves<T, DP>())) void k_attn_bwd_q(AttnParams p, size_t lds_per_wave) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lane_of_wave = lane;
  const int col = lane & 31, hi = lane >> 5;
  const int tid = COOP ? threadIdx.x : lane;
  constexpr int THREADS = COOP ? 64 * kCoopWaves : 64;
  constexpr bool HALF = is_half<T>();
  const uint32_t id = COOP ? blockIdx.x : blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (uint32_t)p.workers * p.heads) return;
  const int head = uniform(id % p.heads), worker = uniform(id / p.heads);
  char* base = lds_raw + (COOP ? 0 : wave * lds_per_wave);
  const AttnLds<T, DP> lds(base);
  float* hist_all = lds.tab + p.n_rel;  // one histogram per wave
  float* hist = hist_all + (COOP ? wave * p.n_rel : 0);
  const bool count = !DELTA && p.part_hist != nullptr;

  const int kv = uniform(head / (p.heads / p.kv_heads));
  const T* kp = (const T*)p.k + kv * p.k_head;
  const T* vp = (const T*)p.v + kv * p.v_head;
  const float slope = p.slope ? p.slope[head] : 0.f, slope2 = slope * kLog2e, scale = p.scale * kLog2e;
  if (p.table) expand_table(lds.tab, p.table + (int64_t)head * p.n_buckets, p.lut, p.n_rel, tid, THREADS);
  if (count)
    for (int i = lane; i < p.n_rel; i += 64) hist[i] = 0.f;
  LongSum dslope, low, high;  // low, high: the two clipped ends of the table

  for (int item = worker; item < p.count; item += p.workers) {
    const AttnWork w = load_work(p.work, item);
    const int mine = (COOP ? wave * kTile : 0) + col;
    const bool live = mine < w.cols;
    const bool busy = (COOP ? wave * kTile : 0) < w.cols;
    const bool whole = (COOP ? wave * kTile : 0) + kTile <= w.cols;
    const int64_t row = (int64_t)w.col0 + (live ? mine : 0);
    const bool once = w.slot < 0 && w.row1 - w.row0 <= kTile;
    if (DELTA && once) continue;

    typename vec8<T>::type qf[DP / 16], df[DP / 16];
    const T* qp = (const T*)p.q + row * p.q_row + head * p.q_head;
    const T* dp_ = (const T*)p.dout + row * p.do_row + head * p.do_head;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      qf[c] = load_col<T>(qp, c * 16 + hi * 8, p.dim, live);
      df[c] = load_col<T>(dp_, c * 16 + hi * 8, p.dim, live);
    }
    const float2 ml = p.stats[head * p.rows_q + row];
    const float ref = ml.x == -INFINITY ? 0.f : ml.x;
    float px = 0, py = 0, pz = 0;
    LongSum gx, gy, gz;
    if (p.slope) px = p.q_pos[3 * row], py = p.q_pos[3 * row + 1], pz = p.q_pos[3 * row + 2];
    int res = 0, res_lo = 0, res_hi = 0;
    if (p.table) {
      res = p.q_res[row];
      column_range(res, res_lo, res_hi);
    }

    f32x16 dq[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dq[d] = acc_zero();
    ColumnScale cs;

    TilePair<T, DP, THREADS> tiles;
    constexpr bool AHEAD = TilePair<T, DP, THREADS>::N <= 8;
    if (AHEAD && w.row0 < w.row1)
      tiles.load(kp + w.row0 * p.k_row, p.k_row, vp + w.row0 * p.v_row, p.v_row, w.row1 - w.row0, p.dim, tid);
    float delta = 0.f, inv_l = 0.f;
    LongSum sum_e, sum_edp;
    if (!DELTA && !once) {
      if (w.slot < 0) {
        const float2 d = p.delta[head * p.rows_q + row];
        delta = d.x, inv_l = d.y;
      } else {
        float e = 0.f, edp = 0.f;
        for (int i = 0; i < w.slots; ++i) {
          const float2 d = p.part_ml[((int64_t)(w.slot0 + (COOP ? wave : 0) + i * w.step) * p.heads + head) * kTile + col];
          if (live) e += d.x, edp += d.y;
        }
        inv_l = e == 0.f ? 0.f : 1.f / e;
        delta = edp * inv_l;
      }
    }
    for (int k0 = w.row0; k0 < w.row1;) {
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
      k0 += kTile;
      if (AHEAD && k0 < w.row1)
        tiles.load(kp + k0 * p.k_row, p.k_row, vp + k0 * p.v_row, p.v_row, w.row1 - k0, p.dim, tid);
      if (!busy) continue;

      const int lane = here(lane_of_wave), col = lane & 31, hi = lane >> 5;
      f32x16 acc = acc_zero(), dp = acc_zero();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c)
        if (c * 16 < p.dim) {
          acc = Mma<T>::run(load_n<T, DP>(lds.a, c, col, hi), qf[c], acc);
          dp = Mma<T>::run(load_n<T, DP>(lds.b, c, col, hi), df[c], dp);
        }
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = acc[r] * scale;
      float far[16];
      if (p.slope) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float4 k = lds.pos[acc_row(r, hi)];
          far[r] = pair_dist(px - k.x, py - k.y, pz - k.z);
          s[r] -= slope2 * far[r];
        }
      }
      int end = -1;
      if (p.table) {
        end = clipped_end(lds.res[col], res_lo, res_hi, 1, p.reach);
        if (end >= 0) {
          const float t = lds.tab[end];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] += t;
        } else {
          float b[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) b[r] = lds.tab[rel_index(lds.res[acc_row(r, hi)], res, p.reach)];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] += b[r];
        }
      }
      if (n < kTile || !whole) {
        const int limit = live ? n : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = acc_row(r, hi) < limit ? s[r] : -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - ref);
      if (DELTA || once) {
        // the sum of exponentials once more, from the very values that D is summed from: then sum_j dS_ij is 0
        float t[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) t[r] = s[r] * dp[r];
        sum_e.add(tile_sum(s));
        sum_edp.add(tile_sum(t));
        if (DELTA) continue;
        const float l = sum_e.both_halves();
        inv_l = l == 0.f ? 0.f : 1.f / l;
        delta = sum_edp.both_halves() * inv_l;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] *= inv_l * (dp[r] - delta);  // dS from here on

      if (p.slope) {
        float ts = 0.f, tx = 0.f, ty = 0.f, tz = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float4 k = lds.pos[acc_row(r, hi)];
          const float dx = px - k.x, dy = py - k.y, dz = pz - k.z;
          ts -= s[r] * far[r];
          const float pull = s[r] * inverse_dist(far[r]);
          tx += pull * dx, ty += pull * dy, tz += pull * dz;
        }
        dslope.add(ts);
        gx.add(tx), gy.add(ty), gz.add(tz);
      }
      if (count && end >= 0) {
        (end ? high : low).add(tile_sum(s));
      } else if (count) {
        // runs of keys of one residue are added up in the lane first; the clipped ends stay in the lane altogether
        float run = 0.f, first_end = 0.f, last_end = 0.f;
        int at = rel_index(lds.res[acc_row(0, hi)], res, p.reach);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          run += s[r];
          const int then = r < 15 ? rel_index(lds.res[acc_row(r < 15 ? r + 1 : 15, hi)], res, p.reach) : -1;
          if (then != at) {
            if (at == 0)
              first_end += run;
            else if (at == 2 * p.reach)
              last_end += run;
            else
              __hip_atomic_fetch_add(hist + at, run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            run = 0.f;
          }
          at = then;
        }
        low.add(first_end);
        high.add(last_end);
      }
      if constexpr (HALF) {
        float largest = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) largest = fmaxf(largest, fabsf(s[r]));
        const float change = cs.follow(fmaxf(largest, other_half(largest)));
        if (__any(change != 1.f)) {
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[d][r] *= change;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= cs.f;
      }
      const Weights<T> s0 = split8<T>(s), s1 = split8<T>(s + 8);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        if (d * 32 >= p.dim) continue;
        tile_mma<T>(dq[d], load_t<T, DP>(lds.a, 0, d * 32, lane, hi), s0, load_t<T, DP>(lds.a, 1, d * 32, lane, hi), s1);
      }
    }

    const int64_t part = ((int64_t)(w.slot + (COOP ? wave : 0)) * p.heads + head) * kTile + col;  // of a piece
    if (DELTA) {
      const float e = sum_e.both_halves(), edp = sum_edp.both_halves(), inv = e == 0.f ? 0.f : 1.f / e;
      if (live && hi == 0) {
        if (w.slot >= 0)
          p.part_ml[part] = make_float2(e, edp);
        else
          p.delta[head * p.rows_q + row] = make_float2(edp * inv, inv);
      }
      continue;
    }
    if (p.part_pos_q) {
      const float x = gx.both_halves(), y = gy.both_halves(), z = gz.both_halves();
      if (live && hi == 0) {
        float* g = w.slot >= 0 ? p.part_g + part * 4 : p.part_pos_q + (head * p.rows_q + row) * 3;
        g[0] = -slope * x, g[1] = -slope * y, g[2] = -slope * z;
      }
    }
    if (live && hi == 0) p.delta[head * p.rows_q + row] = make_float2(delta, inv_l);
    if (live) {
      const float f = HALF ? p.scale / cs.f : p.scale;
      if (w.slot >= 0)
        store_column<float, DP>(p.part_o + part * p.dim, dq, f, p.dim, hi);
      else
        store_column<T, DP>((T*)p.dq + (row * p.heads + head) * p.dim, dq, f, p.dim, hi);
    }
  }

  if (DELTA) return;
  const int64_t part = p.part0 + worker;
  if (p.part_slope) {
    const float sum = wave_sum(dslope.value());
    if (lane == 0) {
      float* out = p.part_slope + (head * (int64_t)p.parts + part) * kCoopWaves;
      if (COOP) {
        out[wave] = sum;
      } else {
        out[0] = sum;
        out[1] = out[2] = out[3] = 0.f;
      }
    }
  }
  if (count) {
    const float first_end = wave_sum(low.value()), last_end = wave_sum(high.value());
    if (lane == 0) {
      hist[0] += first_end;
      hist[2 * p.reach] += last_end;
    }
    tile_sync<COOP>();
    for (int i = tid; i < p.n_rel; i += THREADS) {
      float t = hist_all[i];
      if (COOP)
        for (int k = 1; k < kCoopWaves; ++k) t += hist_all[k * p.n_rel + i];
      p.part_hist[((int64_t)head * p.n_rel + i) * p.parts + part] = t;
    }
  }
}

template <typename T, int DP, bool COOP>
__global__ __launch_bounds__(256, (backward_waves<T, DP>())) void k_attn_bwd_k(AttnParams p, size_t lds_per_wave) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, lane_of_wave = lane;
  const int col = lane & 31, hi = lane >> 5;
  const int tid = COOP ? threadIdx.x : lane;
  constexpr int THREADS = COOP ? 64 * kCoopWaves : 64;
  constexpr bool HALF = is_half<T>();
  const uint32_t id = COOP ? blockIdx.x : blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (uint32_t)p.count * p.kv_heads) return;
  const int kv = uniform(id % p.kv_heads), share = uniform(p.heads / p.kv_heads);
  const AttnWork w = load_work(p.work, uniform(id / p.kv_heads));
  const AttnLds<T, DP> lds(lds_raw + (COOP ? 0 : wave * lds_per_wave));

  const int mine = (COOP ? wave * kTile : 0) + col;
  const bool live = mine < w.cols;
  const bool busy = (COOP ? wave * kTile : 0) < w.cols;
  const bool whole = (COOP ? wave * kTile : 0) + kTile <= w.cols;
  const int64_t row = (int64_t)w.col0 + (live ? mine : 0);

  typename vec8<T>::type kf[DP / 16], vf[DP / 16];
  const T* kp = (const T*)p.k + row * p.k_row + kv * p.k_head;
  const T* vp = (const T*)p.v + row * p.v_row + kv * p.v_head;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    kf[c] = load_col<T>(kp, c * 16 + hi * 8, p.dim, live);
    vf[c] = load_col<T>(vp, c * 16 + hi * 8, p.dim, live);
  }
  float px = 0, py = 0, pz = 0;
  LongSum gx, gy, gz;
  if (p.slope) px = p.k_pos[3 * row], py = p.k_pos[3 * row + 1], pz = p.k_pos[3 * row + 2];
  int res = 0, res_lo = 0, res_hi = 0;
  if (p.table) {
    res = p.k_res[row];
    column_range(res, res_lo, res_hi);
  }

  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d) dk[d] = acc_zero(), dv[d] = acc_zero();
  ColumnScale cs;
  const float scale = p.scale * kLog2e;
  constexpr float PUP = HALF ? 0x1p14f : 1.f;

  for (int sub = 0; sub < share; ++sub) {
    const int head = kv * share + sub;
    const T* qp = (const T*)p.q + head * p.q_head;
    const T* dp_ = (const T*)p.dout + head * p.do_head;
    const float slope = p.slope ? p.slope[head] : 0.f, slope2 = slope * kLog2e;
    if (p.table) {
      tile_sync<COOP>();
      expand_table(lds.tab, p.table + (int64_t)head * p.n_buckets, p.lut, p.n_rel, tid, THREADS);
    }
    TilePair<T, DP, THREADS> tiles;
    constexpr bool AHEAD = TilePair<T, DP, THREADS>::N <= 8;
    if (AHEAD && w.row0 < w.row1)
      tiles.load(qp + w.row0 * p.q_row, p.q_row, dp_ + w.row0 * p.do_row, p.do_row, w.row1 - w.row0, p.dim, tid);
    for (int q0 = w.row0; q0 < w.row1; q0 += kTile) {
      const int n = w.row1 - q0 < kTile ? w.row1 - q0 : kTile;
      if (!AHEAD) tiles.load(qp + q0 * p.q_row, p.q_row, dp_ + q0 * p.do_row, p.do_row, n, p.dim, tid);
      tile_sync<COOP>();
      tiles.store(lds.a, lds.b, n, p.dim, tid);
      if (tid < kTile) {
        const int64_t qr = q0 + (tid < n ? tid : 0);
        if (p.slope) lds.pos[tid] = make_float4(p.q_pos[3 * qr], p.q_pos[3 * qr + 1], p.q_pos[3 * qr + 2], 0.f);
        if (p.table) lds.res[tid] = p.q_res[qr];
        const float top = p.stats[head * p.rows_q + qr].x;
        const float2 d = p.delta[head * p.rows_q + qr];
        lds.stat[tid] = make_float4(top == -INFINITY ? 0.f : top, d.y, d.x, 0.f);
      }
      tile_sync<COOP>();
      const int next = q0 + kTile;
      if (AHEAD && next < w.row1)
        tiles.load(qp + next * p.q_row, p.q_row, dp_ + next * p.do_row, p.do_row, w.row1 - next, p.dim, tid);
      if (!busy) continue;

      const int lane = here(lane_of_wave), col = lane & 31, hi = lane >> 5;
      f32x16 acc = acc_zero(), dp = acc_zero();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c)
        if (c * 16 < p.dim) {
          acc = Mma<T>::run(load_n<T, DP>(lds.a, c, col, hi), kf[c], acc);
          dp = Mma<T>::run(load_n<T, DP>(lds.b, c, col, hi), vf[c], dp);
        }
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = acc[r] * scale;
      float far[16];
      if (p.slope) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float4 q = lds.pos[acc_row(r, hi)];
          far[r] = pair_dist(q.x - px, q.y - py, q.z - pz);
          s[r] -= slope2 * far[r];
        }
      }
      if (p.table) {
        const int end = clipped_end(lds.res[col], res_lo, res_hi, -1, p.reach);
        if (end >= 0) {
          const float t = lds.tab[end];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] += t;
        } else {
          float b[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) b[r] = lds.tab[rel_index(res, lds.res[acc_row(r, hi)], p.reach)];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] += b[r];
        }
      }
      if (n < kTile || !whole) {
        const int limit = live ? n : 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = acc_row(r, hi) < limit ? s[r] : -INFINITY;
      }
      float pr[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float4 st = lds.stat[acc_row(r, hi)];
        const float e = __builtin_amdgcn_exp2f(s[r] - st.x) * st.y;
        s[r] = e * (dp[r] - st.z);  // dS from here on
        pr[r] = e * PUP;
      }
      if (p.part_pos_k) {
        float tx = 0.f, ty = 0.f, tz = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float4 q = lds.pos[acc_row(r, hi)];
          const float dx = q.x - px, dy = q.y - py, dz = q.z - pz;
          const float pull = slope * s[r] * inverse_dist(far[r]);
          tx += pull * dx, ty += pull * dy, tz += pull * dz;
        }
        gx.add(tx), gy.add(ty), gz.add(tz);
      }
      if constexpr (HALF) {
        float largest = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) largest = fmaxf(largest, fabsf(s[r]));
        const float change = cs.follow(fmaxf(largest, other_half(largest)));
        if (__any(change != 1.f)) {
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[d][r] *= change;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= cs.f;
      }
      const Weights<T> s0 = split8<T>(s), s1 = split8<T>(s + 8), p0 = split8<T>(pr), p1 = split8<T>(pr + 8);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        if (d * 32 >= p.dim) continue;
        tile_mma<T>(dv[d], load_t<T, DP>(lds.b, 0, d * 32, lane, hi), p0, load_t<T, DP>(lds.b, 1, d * 32, lane, hi), p1);
        tile_mma<T>(dk[d], load_t<T, DP>(lds.a, 0, d * 32, lane, hi), s0, load_t<T, DP>(lds.a, 1, d * 32, lane, hi), s1);
      }
    }
  }

  const int64_t part = ((int64_t)(w.slot + (COOP ? wave : 0)) * p.kv_heads + kv) * kTile + col;  // of a piece
  if (p.part_pos_k) {
    const float x = gx.both_halves(), y = gy.both_halves(), z = gz.both_halves();
    if (live && hi == 0) {
      float* g = w.slot >= 0 ? p.part_g + part * 4 : p.part_pos_k + (kv * p.rows_k + row) * 3;
      g[0] = x, g[1] = y, g[2] = z;
    }
  }
  if (!live) return;
  const float f = HALF ? p.scale / cs.f : p.scale;
  constexpr float PDOWN = 1.f / PUP;
  if (w.slot >= 0) {
    store_column<float, DP>(p.part_o + part * p.dim, dk, f, p.dim, hi);
    store_column<float, DP>(p.part_o2 + part * p.dim, dv, PDOWN, p.dim, hi);
  } else {
    store_column<T, DP>((T*)p.dk + (row * p.kv_heads + kv) * p.dim, dk, f, p.dim, hi);
    store_column<T, DP>((T*)p.dv + (row * p.kv_heads + kv) * p.dim, dv, PDOWN, p.dim, hi);
  }
}

// Adds up the pieces of a block of columns: one workgroup per (block, head), a thread per four elements of a column.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_bwd_pieces(AttnParams p, int heads, T* out, T* out2, float* pos, int64_t rows) {
  const AttnJoin j = p.join[blockIdx.x];
  const int head = blockIdx.y, quads = p.dim / 4;
  for (int i = threadIdx.x; i < j.cols * quads; i += 256) {
    const int col = i / quads, d = i % quads * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
    for (int s = 0; s < j.slots; ++s) {
      const int64_t at = (((int64_t)(j.slot0 + s * j.step) * heads + head) * kTile + col) * p.dim + d;
      const float4 x = *(const float4*)(p.part_o + at);
      a.x += x.x, a.y += x.y, a.z += x.z, a.w += x.w;
      if (out2) {
        const float4 y = *(const float4*)(p.part_o2 + at);
        b.x += y.x, b.y += y.y, b.z += y.z, b.w += y.w;
      }
    }
    const int64_t to = (((int64_t)j.col0 + col) * heads + head) * p.dim + d;
    store4<T>(out + to, a.x, a.y, a.z, a.w);
    if (out2) store4<T>(out2 + to, b.x, b.y, b.z, b.w);
  }
  if (pos && threadIdx.x < j.cols * 3) {
    const int col = threadIdx.x / 3, c = threadIdx.x % 3;
    float t = 0.f;
    for (int s = 0; s < j.slots; ++s) t += p.part_g[(((int64_t)(j.slot0 + s * j.step) * heads + head) * kTile + col) * 4 + c];
    pos[(head * rows + j.col0 + col) * 3 + c] = t;
  }
}

// Joins the partial sums in a fixed order: positions over heads (a workgroup per work item of the segments), then one
// workgroup per head for its slope and one per (head, bucket) for the table, both summed in float64.
struct AttnPosSegment {
  const AttnWork* work;    // fragments of one or two tiles: their rows (of_rows) or columns, or
  const AttnBlock* block;  // blocks of columns
  int count, of_rows;
  int parts_q, parts_k;  // partial sums of each side that make up the result
  float* out;
};
struct AttnPosJoin {
  AttnPosSegment seg[6];
  int n;
};

__global__ __launch_bounds__(256) void k_attn_bwd_join(AttnParams p, AttnPosJoin join, int n_slope) {
  int b = blockIdx.x;
  const int tid = threadIdx.x;
  for (int i = 0; i < join.n; ++i) {
    const AttnPosSegment g = join.seg[i];
    if (b < g.count) {
      int64_t first, n;
      if (g.work) {
        const AttnWork w = g.work[b];
        first = g.of_rows ? w.row0 : w.col0, n = g.of_rows ? w.row1 - w.row0 : w.cols;
      } else {
        first = g.block[b].col0, n = g.block[b].cols;
      }
      for (int64_t at = first * 3 + tid; at < (first + n) * 3; at += 256) {
        float t = 0.f;
        for (int h = 0; h < g.parts_k; ++h) t += p.part_pos_k[h * p.rows_k * 3 + at];
        for (int h = 0; h < g.parts_q; ++h) t += p.part_pos_q[h * p.rows_q * 3 + at];
        g.out[at] = t;
      }
      return;
    }
    b -= g.count;
  }
  __shared__ double red[4];
  __shared__ int rels[2 * kMaxReach + 1];
  __shared__ int n_rels;
  double t = 0.0;
  float* out;
  if (b < n_slope) {
    const float4* part = (const float4*)(p.part_slope + (int64_t)b * p.parts * kCoopWaves);
    for (int i = tid; i < p.parts; i += 4 * 256) {
      float4 u[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = i + k * 256 < p.parts ? part[i + k * 256] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) t += ((double)u[k].x + u[k].y) + ((double)u[k].z + u[k].w);
    }
    out = p.dslope + b;
  } else {
    const int at = b - n_slope, head = at / p.n_buckets, bucket = at % p.n_buckets;
    if (tid < 64) {  // the differences of this bucket, in their order
      int n = 0;
      for (int base = 0; base < p.n_rel; base += 64) {
        const bool hit = base + tid < p.n_rel && p.lut[base + tid] == bucket;
        const uint64_t mask = __ballot(hit);
        if (hit) rels[n + __popcll(mask & ((1ull << tid) - 1))] = base + tid;
        n += __popcll(mask);
      }
      if (tid == 0) n_rels = n;
    }
    __syncthreads();
    const float* part = p.part_hist + (int64_t)head * p.n_rel * p.parts;
    const int total = n_rels * p.parts;  // (workers() bounds n_rel * parts)
    for (int i = tid; i < total; i += 8 * 256) {
      float u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = i + k * 256;
        u[k] = e < total ? part[(int64_t)rels[e / p.parts] * p.parts + e % p.parts] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) t += u[k];
    }
    out = p.dtable + at;
  }
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if ((tid & 63) == 0) red[tid >> 6] = t;
  __syncthreads();
  if (tid == 0) *out = (float)(red[0] + red[1] + red[2] + red[3]);
}

template <typename T, int DP, bool DELTA>
static int q_launch(const AttnPlanView& by_query, AttnParams p, int lone_workers, int coop_workers, size_t lone_bytes,
                    size_t coop_bytes, hipStream_t st) {
  if (by_query.lone) {
    p.work = by_query.lone_work, p.count = by_query.lone, p.workers = DELTA ? by_query.lone : lone_workers, p.part0 = 0;
    const int64_t total = (int64_t)p.workers * p.heads;
    const int waves = lone_waves(lone_bytes);
    if (!allow_lds((const void*)k_attn_bwd_q<T, DP, false, DELTA>, waves * lone_bytes)) return -5;
    hipLaunchKernelGGL((k_attn_bwd_q<T, DP, false, DELTA>), dim3((unsigned)((total + waves - 1) / waves)),
                       dim3(64 * waves), waves * lone_bytes, st, p, lone_bytes);
  }
  if (by_query.coop) {
    p.work = by_query.coop_work, p.count = by_query.coop, p.workers = DELTA ? by_query.coop : coop_workers;
    p.part0 = lone_workers;
    if (!allow_lds((const void*)k_attn_bwd_q<T, DP, true, DELTA>, coop_bytes)) return -5;
    hipLaunchKernelGGL((k_attn_bwd_q<T, DP, true, DELTA>), dim3((unsigned)((int64_t)p.workers * p.heads)),
                       dim3(64 * kCoopWaves), coop_bytes, st, p, coop_bytes);
  }
  return 0;
}

template <typename T, int DP>
static int bwd_launch(const AttnPlanView& by_query, const AttnPlanView& by_key, AttnParams p, int lone_workers,
                      int coop_workers, hipStream_t st) {
  const int n_rel = p.table ? p.n_rel : 0;
  const size_t tab = AttnLds<T, DP>::bytes(n_rel);
  const size_t lone_q = AttnLds<T, DP>::bytes(n_rel + (p.part_hist ? p.n_rel : 0));
  const size_t coop_q = AttnLds<T, DP>::bytes(n_rel + (p.part_hist ? kCoopWaves * p.n_rel : 0));
  if (by_query.long_rows) {
    const int rc = q_launch<T, DP, true>(by_query, p, lone_workers, coop_workers, tab, tab, st);
    if (rc) return rc;
  }
  const int rc = q_launch<T, DP, false>(by_query, p, lone_workers, coop_workers, lone_q, coop_q, st);
  if (rc) return rc;
  if (by_query.joins) {
    p.join = by_query.join;
    hipLaunchKernelGGL((k_attn_bwd_pieces<T>), dim3(by_query.joins, p.heads), dim3(256), 0, st, p, p.heads, (T*)p.dq,
                       (T*)nullptr, p.part_pos_q, p.rows_q);
  }
  if (by_key.lone) {
    p.work = by_key.lone_work, p.count = by_key.lone;
    const int64_t total = (int64_t)by_key.lone * p.kv_heads;
    const int waves = lone_waves(tab);
    if (!allow_lds((const void*)k_attn_bwd_k<T, DP, false>, waves * tab)) return -5;
    hipLaunchKernelGGL((k_attn_bwd_k<T, DP, false>), dim3((unsigned)((total + waves - 1) / waves)), dim3(64 * waves),
                       waves * tab, st, p, tab);
  }
  if (by_key.coop) {
    p.work = by_key.coop_work, p.count = by_key.coop;
    if (!allow_lds((const void*)k_attn_bwd_k<T, DP, true>, tab)) return -5;
    hipLaunchKernelGGL((k_attn_bwd_k<T, DP, true>), dim3((unsigned)((int64_t)by_key.coop * p.kv_heads)),
                       dim3(64 * kCoopWaves), tab, st, p, tab);
  }
  if (by_key.joins) {
    p.join = by_key.join;
    hipLaunchKernelGGL((k_attn_bwd_pieces<T>), dim3(by_key.joins, p.kv_heads), dim3(256), 0, st, p, p.kv_heads,
                       (T*)p.dk, (T*)p.dv, p.part_pos_k, p.rows_k);
  }
  return 0;
}

static int join_launch(const AttnPlanView& by_query, const AttnPlanView& by_key, const AttnParams& p, int groups,
                       hipStream_t st) {
  AttnPosJoin join = {};
  int64_t blocks = 0;
  auto add = [&](const AttnWork* work, const AttnBlock* block, int count, int of_rows, int parts_q, int parts_k, float* out) {
    if (!count) return;
    join.seg[join.n++] = {work, block, count, of_rows, parts_q, parts_k, out};
    blocks += count;
  };
  if (p.dpos) {
    const bool self = !p.dq_pos;
    add(nullptr, by_key.block, by_key.blocks, 0, self ? p.heads : 0, p.kv_heads, p.dpos);
    add(by_query.pair_work, nullptr, by_query.pair, 1, self ? p.heads : 0, p.kv_heads, p.dpos);
    if (groups > 1) add(by_query.small_work, nullptr, by_query.small, 1, self ? groups : 0, groups, p.dpos);
    if (!self) {
      add(nullptr, by_query.block, by_query.blocks, 0, p.heads, 0, p.dq_pos);
      add(by_query.pair_work, nullptr, by_query.pair, 0, p.heads, 0, p.dq_pos);
      if (groups > 1) add(by_query.small_work, nullptr, by_query.small, 0, groups, 0, p.dq_pos);
    }
  }
  const int n_slope = p.dslope ? p.heads : 0, n_table = p.dtable ? p.heads * p.n_buckets : 0;
  blocks += n_slope + n_table;
  if (blocks) hipLaunchKernelGGL(k_attn_bwd_join, dim3((unsigned)blocks), dim3(256), 0, st, p, join, n_slope);
  return hipGetLastError() == hipSuccess ? 0 : -5;
}

template <typename T>
static int bwd_dim(const AttnPlanView& a, const AttnPlanView& b, const AttnParams& p, int lw, int cw, hipStream_t st) {
  if (p.dim <= 32) return bwd_launch<T, 32>(a, b, p, lw, cw, st);
  if (p.dim <= 64) return bwd_launch<T, 64>(a, b, p, lw, cw, st);
  return bwd_launch<T, 128>(a, b, p, lw, cw, st);
}

int attn_backward(int dtype, const AttnPlanView& by_query, const AttnPlanView& by_key, const AttnParams& p,
                  const AttnWorkers& n, hipStream_t st) {
  int rc = 0;
  switch (dtype) {
    case VSN_F32: rc = bwd_dim<float>(by_query, by_key, p, n.lone, n.coop, st); break;
    case VSN_BF16: rc = bwd_dim<__bf16>(by_query, by_key, p, n.lone, n.coop, st); break;
    default: rc = bwd_dim<_Float16>(by_query, by_key, p, n.lone, n.coop, st); break;
  }
  if (!rc && by_query.pair) {
    AttnParams pair = p;
    pair.work = by_query.pair_work, pair.count = by_query.pair;
    pair.workers = n.pair, pair.part0 = n.lone + n.coop + n.small;
    rc = attn_pair_backward(dtype, pair, st);
  }
  const int groups = small_groups(by_query.small, p.kv_heads);
  if (!rc && by_query.small) {
    AttnParams small = p;
    small.work = by_query.small_work, small.count = by_query.small;
    small.workers = n.small, small.part0 = n.lone + n.coop;
    rc = attn_small(dtype, small, groups, true, st);
  }
  return rc ? rc : join_launch(by_query, by_key, p, groups, st);
}

}  // namespace vsn
