// Fragment attention where one 32 x 32 tile holds a whole fragment (attention.h has the tile): a wave takes a fragment
// and walks its heads.
//
// What does not depend on the head - distances, residue offsets, positions' directions - is computed once per fragment
// and stays in registers; a head's scores are computed once for all of its gradients.  With queries in lanes, dq takes dS
// from the registers; dk and dv contract over the lanes, so dS and P pass through LDS (rounded to the rows' type, as any
// product's operand) and are read back transposed.  The positions' gradient needs only sum_heads slope dS: one pass per
// fragment.  Rows are loaded straight into matrix operands (a lane has its row's 16-byte pieces) and written to LDS from
// there for the products that need them transposed; nothing is read twice.
// Softmax statistics are recomputed: they cost less than reading them.
#include "attention.h"
#include "attention_host.h"

namespace vsn {

constexpr int kPullLd = 33;  // floats per row of the transposed pulls: column reads fall on different banks

template <typename T, int DP>
struct SmallLds {
  static constexpr size_t A = TileShape<T, DP>::BYTES, B = TileShape<T, 32>::BYTES;
  static constexpr size_t PULL = sizeof(float) * kTile * kPullLd;
  static constexpr size_t SCRATCH = A + B > PULL ? A + B : PULL;  // tiles during the heads, pulls after them
  T *a, *b;
  float* pull;
  float4 *kpos, *qpos;
  int* kres;
  float *hist, *slope;  // [heads][n_rel], [heads][64]
  __device__ __forceinline__ SmallLds(char* p, int heads, int n_rel) {
    a = (T*)p;
    b = (T*)(p + A);
    pull = (float*)p;
    kpos = (float4*)(p + ((SCRATCH + 15) & ~(size_t)15));
    qpos = kpos + kTile;
    kres = (int*)(qpos + kTile);
    hist = (float*)(kres + kTile);
    slope = hist + heads * n_rel;
  }
  static size_t bytes(int heads, int n_rel, bool backward) {
    const size_t fixed = ((SCRATCH + 15) & ~(size_t)15) + 2 * kTile * sizeof(float4) + kTile * sizeof(int);
    return (fixed + (backward ? sizeof(float) * heads * (n_rel + 64) : 0) + 15) & ~(size_t)15;
  }
};

// a lane's row of a tile, from the pieces it holds as an operand
template <typename T, int DP>
__device__ __forceinline__ void put_rows(T* tile, const typename vec8<T>::type (&f)[DP / 16], int col, int hi) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c)
    *(typename vec8<T>::type*)(tile + col * TileShape<T, DP>::LD + c * 16 + hi * 8) = f[c];
}
// the lane's 16 values as its row of [column][row]
template <typename T>
__device__ __forceinline__ void put_scores(T* tile, const float* v, int col, int hi) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
    store4<T>(tile + col * TileShape<T, 32>::LD + 8 * g + 4 * hi, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
}

// distances (units of the input) and reciprocals, table indices, from LDS
struct SmallGeometry {
  float far[16], inv[16];
  int at[16];
};

template <typename T, int DP, bool BACKWARD>
__device__ __forceinline__ void small_geometry(const AttnParams& p, const AttnWork& w, const SmallLds<T, DP>& lds,
                                               SmallGeometry& g, int nk, int64_t q_row, int lane, int col, int hi) {
  tile_sync<false>();
  if (lane < kTile) {
    const int64_t kr = (int64_t)w.row0 + (col < nk ? col : 0);
    if (p.slope) {
      lds.kpos[col] = nk ? make_float4(p.k_pos[3 * kr], p.k_pos[3 * kr + 1], p.k_pos[3 * kr + 2], 0.f)
                         : make_float4(0.f, 0.f, 0.f, 0.f);
      if (w.cols) lds.qpos[col] = make_float4(p.q_pos[3 * q_row], p.q_pos[3 * q_row + 1], p.q_pos[3 * q_row + 2], 0.f);
    }
    if (p.table) lds.kres[col] = nk ? p.k_res[kr] : 0;
  }
  tile_sync<false>();
  if (p.slope) {
    const float4 q = w.cols ? lds.qpos[col] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float4 k = lds.kpos[acc_row(r, hi)];
      g.far[r] = pair_dist(q.x - k.x, q.y - k.y, q.z - k.z, g.inv[r]);
    }
  }
  if (p.table) {
    const int res = w.cols ? p.q_res[q_row] : 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) g.at[r] = rel_index(lds.kres[acc_row(r, hi)], res, p.reach);
  }
}

// the scores of one head, masked, from the product q.k
template <typename T>
__device__ __forceinline__ void small_scores(const AttnParams& p, const SmallGeometry& g, const f32x16& acc, float scale,
                                             float slope2, const float* tab, int limit, int hi, float* s) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = acc[r] * scale;
  if (p.slope) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] -= slope2 * g.far[r];
  }
  if (p.table) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] += tab[g.at[r]];
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = acc_row(r, hi) < limit ? s[r] : -INFINITY;
}

// s -> exponentials; returns the maximum
__device__ __forceinline__ float small_exp(float* s) {
  float top = s[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
  top = fmaxf(top, other_half(top));
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] - ref);
  return top;
}

template <typename T, int DP>
__global__ __launch_bounds__(256) void k_attn_small_fwd(AttnParams p, size_t per_wave, int groups) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, hi = lane >> 5;
  float* tab = (float*)lds_raw;  // [heads][n_rel]
  const int n_rel = p.table ? p.n_rel : 0;
  for (int i = threadIdx.x; i < p.heads * n_rel; i += blockDim.x)
    tab[i] = table_log2(p.table[(int64_t)(i / n_rel) * p.n_buckets + p.lut[i % n_rel]]);
  __syncthreads();
  const int64_t id = (int64_t)blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (int64_t)p.count * groups) return;
  const SmallLds<T, DP> lds(lds_raw + ((sizeof(float) * p.heads * n_rel + 15) & ~(size_t)15) + wave * per_wave, p.heads, 0);
  const AttnWork w = p.work[id / groups];
  const int nq = w.cols, nk = w.row1 - w.row0;
  const bool live = col < nq;
  const int64_t q_row = (int64_t)w.col0 + (live ? col : 0), k_row = (int64_t)w.row0 + (col < nk ? col : 0);
  SmallGeometry g;
  small_geometry<T, DP, false>(p, w, lds, g, nk, q_row, lane, col, hi);
  const float scale = p.scale * kLog2e;
  const int share = p.heads / p.kv_heads, each = p.heads / groups, h0 = (int)(id % groups) * each;
  for (int head = h0; head < h0 + each; ++head) {
    const int kv = head / share;
    typename vec8<T>::type qf[DP / 16], kf[DP / 16], vf[DP / 16];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      qf[c] = load_col<T>((const T*)p.q + q_row * p.q_row + head * p.q_head, c * 16 + hi * 8, p.dim, live);
      kf[c] = load_col<T>((const T*)p.k + k_row * p.k_row + kv * p.k_head, c * 16 + hi * 8, p.dim, col < nk);
      vf[c] = load_col<T>((const T*)p.v + k_row * p.v_row + kv * p.v_head, c * 16 + hi * 8, p.dim, col < nk);
    }
    f32x16 acc = acc_zero();
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
      if (c * 16 < p.dim) acc = Mma<T>::run(kf[c], qf[c], acc);
    tile_sync<false>();
    put_rows<T, DP>(lds.a, vf, col, hi);
    tile_sync<false>();
    float s[16];
    small_scores<T>(p, g, acc, scale, p.slope ? p.slope[head] * kLog2e : 0.f, tab + head * n_rel, live ? nk : 0, hi, s);
    const float top = small_exp(s);
    float l = tile_sum(s);
    l += other_half(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const typename vec8<T>::type p0 = pack8<T>(s), p1 = pack8<T>(s + 8);
    if (live && hi == 0 && p.stats) p.stats[head * p.rows_q + q_row] = make_float2(top, l);
    T* op = (T*)p.out + q_row * p.out_row + head * p.out_head;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      if (d * 32 >= p.dim) continue;
      f32x16 o = acc_zero();
      o = Mma<T>::run(load_t<T, DP>(lds.a, 0, d * 32, lane, hi), p0, o);
      o = Mma<T>::run(load_t<T, DP>(lds.a, 1, d * 32, lane, hi), p1, o);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = d * 32 + 8 * k + 4 * hi;
        if (live && e < p.dim) store4<T>(op + e, o[4 * k] * inv, o[4 * k + 1] * inv, o[4 * k + 2] * inv, o[4 * k + 3] * inv);
      }
    }
  }
}

// groups: 1 (a wave walks all heads and writes the positions' gradient), or kv_heads (a wave takes the heads of one key
// head, where there are few fragments; the positions' gradients are joined afterwards)
template <typename T, int DP>
__global__ __launch_bounds__(256) void k_attn_small_bwd(AttnParams p, size_t per_wave, int groups) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  constexpr bool HALF = sizeof(T) == 2 && !__is_same(T, __bf16);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, hi = lane >> 5;
  float* tab = (float*)lds_raw;
  const int n_rel = p.table ? p.n_rel : 0;
  for (int i = threadIdx.x; i < p.heads * n_rel; i += blockDim.x)
    tab[i] = table_log2(p.table[(int64_t)(i / n_rel) * p.n_buckets + p.lut[i % n_rel]]);
  __syncthreads();
  const int64_t id = (int64_t)blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (int64_t)p.workers * groups) return;
  const SmallLds<T, DP> lds(lds_raw + ((sizeof(float) * p.heads * n_rel + 15) & ~(size_t)15) + wave * per_wave, p.heads, n_rel);
  const int worker = (int)(id / groups), group = (int)(id % groups);
  const int share = p.heads / p.kv_heads, each = p.heads / groups, h0 = group * each;
  for (int i = lane; i < p.heads * n_rel; i += 64) lds.hist[i] = 0.f;
  for (int i = lane; i < p.heads * 64; i += 64) lds.slope[i] = 0.f;
  const float scale = p.scale * kLog2e;

  for (int item = worker; item < p.count; item += p.workers) {
    const AttnWork w = p.work[item];
    const int nq = w.cols, nk = w.row1 - w.row0;
    const bool live = col < nq, key = col < nk;
    const int64_t q_row = (int64_t)w.col0 + (live ? col : 0), k_row = (int64_t)w.row0 + (key ? col : 0);
    SmallGeometry g;
    small_geometry<T, DP, true>(p, w, lds, g, nk, q_row, lane, col, hi);
    float weight[16];  // sum over heads of slope dS
#pragma unroll
    for (int r = 0; r < 16; ++r) weight[r] = 0.f;
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dk[d] = acc_zero(), dv[d] = acc_zero();

    for (int head = h0; head < h0 + each; ++head) {
      const int kv = head / share;
      typename vec8<T>::type qf[DP / 16], df[DP / 16], kf[DP / 16], vf[DP / 16];
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        qf[c] = load_col<T>((const T*)p.q + q_row * p.q_row + head * p.q_head, c * 16 + hi * 8, p.dim, live);
        kf[c] = load_col<T>((const T*)p.k + k_row * p.k_row + kv * p.k_head, c * 16 + hi * 8, p.dim, key);
        df[c] = load_col<T>((const T*)p.dout + q_row * p.do_row + head * p.do_head, c * 16 + hi * 8, p.dim, live);
        vf[c] = load_col<T>((const T*)p.v + k_row * p.v_row + kv * p.v_head, c * 16 + hi * 8, p.dim, key);
      }
      f32x16 acc = acc_zero(), dp = acc_zero();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c)
        if (c * 16 < p.dim) {
          acc = Mma<T>::run(kf[c], qf[c], acc);
          dp = Mma<T>::run(vf[c], df[c], dp);
        }
      const float slope = p.slope ? p.slope[head] : 0.f;
      float s[16], t[16];
      small_scores<T>(p, g, acc, scale, slope * kLog2e, tab + head * n_rel, live ? nk : 0, hi, s);
      small_exp(s);
#pragma unroll
      for (int r = 0; r < 16; ++r) t[r] = s[r] * dp[r];
      float l = tile_sum(s), delta = tile_sum(t);
      l += other_half(l);
      delta += other_half(delta);
      const float inv_l = l == 0.f ? 0.f : 1.f / l;
      delta *= inv_l;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] *= inv_l;                // P
        t[r] = s[r] * (dp[r] - delta);  // dS
      }
      if (p.slope) {
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          sum -= t[r] * g.far[r];
          weight[r] += slope * t[r];
        }
        lds.slope[head * 64 + lane] += sum;
      }
      if (p.part_hist) {
        float run = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {  // (runs of keys of one residue are added up in the lane first)
          run += t[r];
          if (r == 15 || g.at[r < 15 ? r + 1 : 15] != g.at[r]) {
            __hip_atomic_fetch_add(lds.hist + head * n_rel + g.at[r], run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            run = 0.f;
          }
        }
      }
      // float16: the largest |dS| of the tile to 2^14, P times 2^14
      float up = 1.f, down = 1.f;
      constexpr float PUP = HALF ? 0x1p14f : 1.f;
      if constexpr (HALF) {
        float largest = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) largest = fmaxf(largest, fabsf(t[r]));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor(largest, o, 64));
        if (largest >= 0x1p-80f && largest < INFINITY) {
          up = ldexpf(1.f, 14 - ilogbf(largest));
          down = ldexpf(1.f, ilogbf(largest) - 14);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) t[r] *= up, s[r] *= PUP;
      }
      tile_sync<false>();
      put_rows<T, DP>(lds.a, df, col, hi);
      put_scores<T>(lds.b, s, col, hi);
      tile_sync<false>();
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
        if (d * 32 < p.dim)
          tile_mma<T>(dv[d], load_t<T, DP>(lds.a, 0, d * 32, lane, hi), load_t<T, 32>(lds.b, 0, 0, lane, hi),
                      load_t<T, DP>(lds.a, 1, d * 32, lane, hi), load_t<T, 32>(lds.b, 1, 0, lane, hi));
      tile_sync<false>();
      put_rows<T, DP>(lds.a, qf, col, hi);
      put_scores<T>(lds.b, t, col, hi);
      tile_sync<false>();
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        if (d * 32 >= p.dim) continue;
        f32x16 x = acc_zero();
        x = Mma<T>::run(load_t<T, DP>(lds.a, 0, d * 32, lane, hi), load_t<T, 32>(lds.b, 0, 0, lane, hi), x);
        x = Mma<T>::run(load_t<T, DP>(lds.a, 1, d * 32, lane, hi), load_t<T, 32>(lds.b, 1, 0, lane, hi), x);
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] += x[r] * down;
      }
      tile_sync<false>();
      put_rows<T, DP>(lds.a, kf, col, hi);
      tile_sync<false>();
      const typename vec8<T>::type t0 = pack8<T>(t), t1 = pack8<T>(t + 8);
      const float f = p.scale * down;
      T* oq = (T*)p.dq + (q_row * p.heads + head) * p.dim;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        if (d * 32 >= p.dim) continue;
        f32x16 x = acc_zero();
        x = Mma<T>::run(load_t<T, DP>(lds.a, 0, d * 32, lane, hi), t0, x);
        x = Mma<T>::run(load_t<T, DP>(lds.a, 1, d * 32, lane, hi), t1, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = d * 32 + 8 * k + 4 * hi;
          if (live && e < p.dim) store4<T>(oq + e, x[4 * k] * f, x[4 * k + 1] * f, x[4 * k + 2] * f, x[4 * k + 3] * f);
        }
      }
      if (head % share == share - 1) {
        constexpr float PDOWN = 1.f / PUP;
        T* ok = (T*)p.dk + (k_row * p.kv_heads + kv) * p.dim;
        T* ov = (T*)p.dv + (k_row * p.kv_heads + kv) * p.dim;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int e = d * 32 + 8 * k + 4 * hi;
            if (!key || e >= p.dim) continue;
            store4<T>(ok + e, dk[d][4 * k] * p.scale, dk[d][4 * k + 1] * p.scale, dk[d][4 * k + 2] * p.scale, dk[d][4 * k + 3] * p.scale);
            store4<T>(ov + e, dv[d][4 * k] * PDOWN, dv[d][4 * k + 1] * PDOWN, dv[d][4 * k + 2] * PDOWN, dv[d][4 * k + 3] * PDOWN);
          }
          dk[d] = acc_zero(), dv[d] = acc_zero();
        }
      }
    }

    if (p.dpos) {
      // w_ij = sum_heads slope dS / r: the query's share in its lane, the key's after a pass through LDS
      const float4 q = lds.qpos[col];
      float x = 0.f, y = 0.f, z = 0.f;
      tile_sync<false>();
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = acc_row(r, hi);
        const float4 k = lds.kpos[row];
        const float f = live ? weight[r] * g.inv[r] : 0.f;
        x -= f * (q.x - k.x), y -= f * (q.y - k.y), z -= f * (q.z - k.z);
        lds.pull[col * kPullLd + row] = f;
      }
      tile_sync<false>();
      const float4 k = lds.kpos[col];
      float u = 0.f, v = 0.f, t = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = acc_row(r, hi);
        if (row < nq) {
          const float4 o = lds.qpos[row];
          const float f = lds.pull[row * kPullLd + col];
          u += f * (o.x - k.x), v += f * (o.y - k.y), t += f * (o.z - k.z);
        }
      }
      x += other_half(x), y += other_half(y), z += other_half(z);
      u += other_half(u), v += other_half(v), t += other_half(t);
      if (hi == 0) {
        if (groups == 1 && !p.dq_pos) {  // queries and keys are the same rows
          if (key) p.dpos[3 * k_row] = x + u, p.dpos[3 * k_row + 1] = y + v, p.dpos[3 * k_row + 2] = z + t;
        } else {
          float* gq = groups == 1 ? p.dq_pos + 3 * q_row : p.part_pos_q + (group * p.rows_q + q_row) * 3;
          float* gk = groups == 1 ? p.dpos + 3 * k_row : p.part_pos_k + (group * p.rows_k + k_row) * 3;
          if (live) gq[0] = x, gq[1] = y, gq[2] = z;
          if (key) gk[0] = u, gk[1] = v, gk[2] = t;
        }
      }
    }
  }

  tile_sync<false>();
  const int64_t part = p.part0 + worker;
  for (int head = h0; head < h0 + each; ++head) {
    if (p.part_slope) {
      const float sum = wave_sum(lds.slope[head * 64 + lane]);
      if (lane < kCoopWaves) p.part_slope[(head * (int64_t)p.parts + part) * kCoopWaves + lane] = lane ? 0.f : sum;
    }
    if (p.part_hist)
      for (int i = lane; i < n_rel; i += 64) p.part_hist[((int64_t)head * n_rel + i) * p.parts + part] = lds.hist[head * n_rel + i];
  }
}

template <typename T, int DP>
static int small_launch(AttnParams p, int groups, bool backward, hipStream_t st) {
  const int n_rel = p.table ? p.n_rel : 0;
  const size_t tab = (sizeof(float) * p.heads * n_rel + 15) & ~(size_t)15;
  const size_t bytes = SmallLds<T, DP>::bytes(p.heads, n_rel, backward);
  const int64_t total = (int64_t)(backward ? p.workers : p.count) * groups;
  int waves = total <= 1024 ? 1 : 4;
  while (waves > 1 && tab + waves * bytes > kLdsPerCu / 2) waves /= 2;
  const size_t lds = tab + waves * bytes;
  const dim3 grid((unsigned)((total + waves - 1) / waves)), block(64 * waves);
  if (backward) {
    if (!allow_lds((const void*)k_attn_small_bwd<T, DP>, lds)) return -5;
    hipLaunchKernelGGL((k_attn_small_bwd<T, DP>), grid, block, lds, st, p, bytes, groups);
  } else {
    if (!allow_lds((const void*)k_attn_small_fwd<T, DP>, lds)) return -5;
    hipLaunchKernelGGL((k_attn_small_fwd<T, DP>), grid, block, lds, st, p, bytes, groups);
  }
  return 0;
}

template <typename T>
static int small_dim(const AttnParams& p, int groups, bool backward, hipStream_t st) {
  if (p.dim <= 32) return small_launch<T, 32>(p, groups, backward, st);
  if (p.dim <= 64) return small_launch<T, 64>(p, groups, backward, st);
  return small_launch<T, 128>(p, groups, backward, st);
}

int attn_small(int dtype, const AttnParams& p, int groups, bool backward, hipStream_t st) {
  switch (dtype) {
    case VSN_F32: return small_dim<float>(p, groups, backward, st);
    case VSN_BF16: return small_dim<__bf16>(p, groups, backward, st);
    default: return small_dim<_Float16>(p, groups, backward, st);
  }
}

}  // namespace vsn
