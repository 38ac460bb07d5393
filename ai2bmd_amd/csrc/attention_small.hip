// Fragment attention where one 32 x 32 tile holds a whole fragment (attention.h has the tile): a wave takes a fragment
// and walks its heads.
//
// What does not depend on the head - distances, residue offsets, positions' directions - is computed once per fragment
// and stays in registers; a head's scores are computed once for all of its gradients.  With queries in lanes, dq takes dS
// from the registers; dk and dv contract over the lanes, so dS and P pass through LDS (in two parts of 16-bit rows' type, as
// any product's weights) and are read back transposed.  The positions' gradient needs only sum_heads slope dS: one pass per
// fragment.  Rows are loaded straight into matrix operands (a lane has its row's 16-byte pieces) and written to LDS from
// there for the products that need them transposed; nothing is read twice.
// Softmax statistics are recomputed: they cost less than reading them.
// 3600 fragments of 12 ... 32 atoms, 8 heads of 32: float32 forward 77 us (3.7 TB/s), backward 162 us (3.1 TB/s); bf16 forward
// 51 us, backward with the table 127 us.  Bound by one wave's chain of products, exchanges and LDS passes per head, of which
// registers allow two waves per SIMD; the next head's rows are on their way meanwhile.
#include "attention.h"
#include "attention_host.h"

namespace vsn {

// Waves per SIMD that the backward kernel is compiled for; registers are what limits them.  4096 fragments, heads of 32, both
// directions at one, two and three (spilling): float32 440, 407 and 688 us, bf16 with the table 323, 323 and 409 us.
template <typename T, int DP>
constexpr int small_waves() {
  return DP > 64 || (DP > 32 && sizeof(T) == 4) ? 1 : 2;
}

constexpr int kPullLd = 33;  // floats per row of the transposed pulls: column reads fall on different banks

// The lane's 16 weights as its row of [column][row], 16-bit rows' second parts in a tile behind the first; and a product's
// operand of rows 16 c ... + 15, read back transposed.
template <typename T>
struct WeightTile {
  static constexpr int AT = TileShape<T, 32>::LD * kTile;  // of the second parts
  static constexpr size_t BYTES = (sizeof(T) == 2 ? 2 : 1) * TileShape<T, 32>::BYTES;
  static __device__ __forceinline__ void put(T* tile, const Weights<T>& a, const Weights<T>& b, int col, int hi) {
    T* row = tile + col * TileShape<T, 32>::LD + 4 * hi;
    put8(row, a.hi);
    put8(row + 16, b.hi);
    if constexpr (sizeof(T) == 2) {
      put8(row + AT, a.lo);
      put8(row + AT + 16, b.lo);
    }
  }
  static __device__ __forceinline__ Weights<T> get(const T* tile, int c, int lane, int hi) {
    Weights<T> w;
    w.hi = load_t<T, 32>(tile, c, 0, lane, hi);
    if constexpr (sizeof(T) == 2) w.lo = load_t<T, 32>(tile + AT, c, 0, lane, hi);
    return w;
  }

 private:
  static __device__ __forceinline__ void put8(T* row, const typename vec8<T>::type& v) {
    typedef T half4 __attribute__((ext_vector_type(4)));
    *(half4*)row = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    *(half4*)(row + 8) = __builtin_shufflevector(v, v, 4, 5, 6, 7);
  }
};

template <typename T, int DP>
struct SmallLds {
  static constexpr size_t A = TileShape<T, DP>::BYTES, B = WeightTile<T>::BYTES;
  static constexpr size_t PULL = sizeof(float) * kTile * kPullLd;
  T *dout, *q, *k;  // rows to be read transposed (the forward pass has v in `dout`)
  T* score;         // [query][key]: P, then dS
  float* pull;      // after the heads, in the tiles' place
  float4 *kpos, *qpos;
  int* kres;
  float* hist;  // [heads][n_rel]
  __device__ __forceinline__ SmallLds(char* p, bool backward) {
    dout = (T*)p;
    q = (T*)(p + A);
    k = (T*)(p + 2 * A);
    score = (T*)(p + 3 * A);
    pull = (float*)p;
    kpos = (float4*)(p + scratch(backward));
    qpos = kpos + kTile;
    kres = (int*)(qpos + kTile);
    hist = (float*)(kres + kTile);
  }
  static constexpr __host__ __device__ size_t scratch(bool backward) {
    return ((backward ? (3 * A + B > PULL ? 3 * A + B : PULL) : A) + 15) & ~(size_t)15;
  }
  static size_t bytes(int heads, int n_rel, bool backward) {
    return (scratch(backward) + 2 * kTile * sizeof(float4) + kTile * sizeof(int) +
            (backward ? sizeof(float) * heads * n_rel : 0) + 15) & ~(size_t)15;
  }
};

// a lane's row of a tile, from the pieces it holds as an operand
template <typename T, int DP>
__device__ __forceinline__ void put_rows(T* tile, const typename vec8<T>::type (&f)[DP / 16], int col, int hi) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c)
    *(typename vec8<T>::type*)(tile + col * TileShape<T, DP>::LD + c * 16 + hi * 8) = f[c];
}
// A lane's row, loaded without a branch: the row is one of the fragment's in any case, a column beyond the end is
// another one of it.  Both are zeroed where the row is used (keep_rows), so that nothing waits for a load ahead of that.
// `base` is the wave's (its fragment's first row), `lane` the lane's offset in elements.
template <typename T, int DP>
__device__ __forceinline__ void load_rows(typename vec8<T>::type (&f)[DP / 16], const T* base, uint32_t lane, int dim,
                                          int hi) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c)
    f[c] = *(const typename vec8<T>::type*)(base + (lane + (c * 16 + hi * 8 < dim ? c * 16 + hi * 8 : 0)));
}
template <typename T, int DP>
__device__ __forceinline__ void keep_rows(typename vec8<T>::type (&f)[DP / 16], int dim, int hi, bool live) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    typename vec8<T>::type zero;
#pragma unroll
    for (int i = 0; i < 8; ++i) zero[i] = (T)0.f;
    f[c] = live && c * 16 + hi * 8 < dim ? f[c] : zero;
  }
}
// distances and table indices of the lane's 16 pairs
struct SmallGeometry {
  float far[16];
  uint32_t pair[8];  // two table indices each
  // (unpacked where it is used: 16 indices kept over the heads would cost a wave per SIMD)
  __device__ __forceinline__ void here() {
#pragma unroll
    for (int i = 0; i < 8; ++i) compute_here(pair[i]);
  }
  __device__ __forceinline__ int at(int r) const { return r & 1 ? pair[r >> 1] >> 16 : pair[r >> 1] & 0xffff; }
};

template <typename T, int DP>
__device__ __forceinline__ void small_geometry(const AttnParams& p, const AttnWork& w, const SmallLds<T, DP>& lds,
                                               SmallGeometry& g, int nk, int64_t q_row, int lane, int col, int hi) {
  tile_sync<false>();
  if (lane < kTile) {
    const int64_t kr = (int64_t)w.row0 + (col < nk ? col : 0);
    if (p.slope) {
      lds.kpos[col] = make_float4(p.k_pos[3 * kr], p.k_pos[3 * kr + 1], p.k_pos[3 * kr + 2], 0.f);
      lds.qpos[col] = make_float4(p.q_pos[3 * q_row], p.q_pos[3 * q_row + 1], p.q_pos[3 * q_row + 2], 0.f);
    }
    if (p.table) lds.kres[col] = p.k_res[kr];
  }
  tile_sync<false>();
  if (p.slope) {
    const float4 q = lds.qpos[col];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float4 k = lds.kpos[acc_row(r, hi)];
      g.far[r] = pair_dist(q.x - k.x, q.y - k.y, q.z - k.z);
    }
  }
  if (p.table) {
    const int res = p.q_res[q_row];
#pragma unroll
    for (int r = 0; r < 16; r += 2)
      g.pair[r >> 1] = rel_index(lds.kres[acc_row(r, hi)], res, p.reach) |
                       rel_index(lds.kres[acc_row(r + 1, hi)], res, p.reach) << 16;
  }
}

// the scores of one head, masked, from the product q.k
template <typename T>
__device__ __forceinline__ void small_scores(const AttnParams& p, SmallGeometry& g, const f32x16& acc, float scale,
                                             float slope2, const float* tab, int limit, int hi, float* s) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = acc[r] * scale;
  if (p.slope) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] -= slope2 * g.far[r];
  }
  if (p.table) {
    g.here();
    float b[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) b[r] = tab[g.at(r)];
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] += b[r];
  }
  compute_here(limit);
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = acc_row(r, hi) < limit ? s[r] : -INFINITY;
}

// s -> exponentials relative to exp_ref of their maximum; returns that
template <typename T>
__device__ __forceinline__ float small_exp(float* s) {
  float top = s[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
  top = exp_ref<T>(fmaxf(top, other_half(top)));
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
  for (int h = 0; n_rel && h < p.heads; ++h)
    expand_table(tab + h * n_rel, p.table + (int64_t)h * p.n_buckets, p.lut, n_rel, threadIdx.x, blockDim.x);
  float* slopes = tab + p.heads * n_rel;  // [heads]
  for (int i = threadIdx.x; i < p.heads; i += blockDim.x) slopes[i] = p.slope ? p.slope[i] : 0.f;
  __syncthreads();
  const uint32_t id = blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (uint32_t)p.count * groups) return;
  const SmallLds<T, DP> lds(lds_raw + ((sizeof(float) * p.heads * (n_rel + 1) + 15) & ~(size_t)15) + wave * per_wave, false);
  const AttnWork w = load_work(p.work, uniform(id / groups));
  const int nq = w.cols, nk = w.row1 - w.row0;
  const bool live = col < nq;
  const int64_t q_row = (int64_t)w.col0 + (live ? col : 0);
  SmallGeometry g;
  small_geometry<T, DP>(p, w, lds, g, nk, q_row, lane, col, hi);
  const float scale = p.scale * kLog2e;
  const int share = uniform(p.heads / p.kv_heads), each = uniform(p.heads / groups), h0 = uniform(id % groups) * each;
  const uint32_t q_at = (live ? col : 0) * (uint32_t)p.q_row;
  const uint32_t k_at = (col < nk ? col : 0) * (uint32_t)p.k_row, v_at = (col < nk ? col : 0) * (uint32_t)p.v_row;
  const int lane_of_item = lane;
  typename vec8<T>::type qf[DP / 16], kf[DP / 16], vf[DP / 16];
  auto load = [&](int head) {
    const int kv = uniform(head / share);
    load_rows<T, DP>(qf, (const T*)p.q + w.col0 * p.q_row + head * p.q_head, q_at, p.dim, hi);
    load_rows<T, DP>(kf, (const T*)p.k + w.row0 * p.k_row + kv * p.k_head, k_at, p.dim, hi);
    load_rows<T, DP>(vf, (const T*)p.v + w.row0 * p.v_row + kv * p.v_head, v_at, p.dim, hi);
  };
  load(h0);
  for (int head = h0; head < h0 + each; ++head) {
    const int lane = here(lane_of_item), col = lane & 31, hi = lane >> 5;
    keep_rows<T, DP>(qf, p.dim, hi, live);
    keep_rows<T, DP>(kf, p.dim, hi, col < nk);
    keep_rows<T, DP>(vf, p.dim, hi, col < nk);
    f32x16 acc = acc_zero();
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
      if (c * 16 < p.dim) acc = Mma<T>::run(kf[c], qf[c], acc);
    tile_sync<false>();
    put_rows<T, DP>(lds.dout, vf, col, hi);
    tile_sync<false>();
    if (head + 1 < h0 + each) load(head + 1);  // in flight while this head is computed
    float s[16];
    small_scores<T>(p, g, acc, scale, slopes[head] * kLog2e, tab + head * n_rel, live ? nk : 0, hi, s);
    const float ref = small_exp<T>(s);
    float l = tile_sum(s);
    l += other_half(l);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const Weights<T> p0 = split8<T>(s), p1 = split8<T>(s + 8);
    if (live && hi == 0 && p.stats) p.stats[head * p.rows_q + q_row] = attn_stats<T>(ref, l);
    T* op = (T*)p.out + w.col0 * p.out_row + head * p.out_head;
    const uint32_t o_at = col * (uint32_t)p.out_row;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      if (d * 32 >= p.dim) continue;
      f32x16 o = acc_zero();
      o = mma<T>(load_t<T, DP>(lds.dout, 0, d * 32, lane, hi), p0, o);
      if (nk > 16) o = mma<T>(load_t<T, DP>(lds.dout, 1, d * 32, lane, hi), p1, o);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = d * 32 + 8 * k + 4 * hi;
        if (live && e < p.dim) store4<T>(op + (o_at + e), o[4 * k] * inv, o[4 * k + 1] * inv, o[4 * k + 2] * inv, o[4 * k + 3] * inv);
      }
    }
  }
}

// groups: 1 (a wave walks all heads and writes the positions' gradient), or kv_heads (a wave takes the heads of one key
// head, where there are few fragments; the positions' gradients are joined afterwards)
template <typename T, int DP, bool SHARE>
__global__ __launch_bounds__(256, (small_waves<T, DP>())) void k_attn_small_bwd(AttnParams p, size_t per_wave, int groups) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  constexpr bool HALF = is_half<T>();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane_of_wave = threadIdx.x & 63;
  float* tab = (float*)lds_raw;
  const int n_rel = p.table ? p.n_rel : 0;
  for (int h = 0; n_rel && h < p.heads; ++h)
    expand_table(tab + h * n_rel, p.table + (int64_t)h * p.n_buckets, p.lut, n_rel, threadIdx.x, blockDim.x);
  float* slopes = tab + p.heads * n_rel;  // [heads]
  for (int i = threadIdx.x; i < p.heads; i += blockDim.x) slopes[i] = p.slope ? p.slope[i] : 0.f;
  __syncthreads();
  const uint32_t id = blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (uint32_t)p.workers * groups) return;
  const SmallLds<T, DP> lds(lds_raw + ((sizeof(float) * p.heads * (n_rel + 1) + 15) & ~(size_t)15) + wave * per_wave, true);
  const int worker = uniform(id / groups), group = uniform(id % groups);
  const int share = SHARE ? uniform(p.heads / p.kv_heads) : 1, each = uniform(p.heads / groups), h0 = group * each;
  for (int i = lane_of_wave; i < p.heads * n_rel; i += 64) lds.hist[i] = 0.f;
  float dslope = 0.f;  // of head `lane`
  const float scale = p.scale * kLog2e;

  for (int item = worker; item < p.count; item += p.workers) {
    const AttnWork w = load_work(p.work, item);
    const int lane = here(lane_of_wave), col = lane & 31, hi = lane >> 5;
    const int nq = w.cols, nk = w.row1 - w.row0;
    const bool live = col < nq, key = col < nk;
    const int64_t q_row = (int64_t)w.col0 + (live ? col : 0), k_row = (int64_t)w.row0 + (key ? col : 0);
    SmallGeometry g;
    small_geometry<T, DP>(p, w, lds, g, nk, q_row, lane, col, hi);
    float weight[16];  // sum over heads of slope dS
#pragma unroll
    for (int r = 0; r < 16; ++r) weight[r] = 0.f;
    f32x16 dk[DP / 32], dv[DP / 32];  // over the heads that share a key head
    if (SHARE)
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) dk[d] = acc_zero(), dv[d] = acc_zero();

    const uint32_t q_at = (live ? col : 0) * (uint32_t)p.q_row, d_at = (live ? col : 0) * (uint32_t)p.do_row;
    const uint32_t k_at = (key ? col : 0) * (uint32_t)p.k_row, v_at = (key ? col : 0) * (uint32_t)p.v_row;
    typename vec8<T>::type qf[DP / 16], df[DP / 16], kf[DP / 16], vf[DP / 16];
    auto load = [&](int head) {
      const int kv = SHARE ? uniform(head / share) : head;
      load_rows<T, DP>(qf, (const T*)p.q + w.col0 * p.q_row + head * p.q_head, q_at, p.dim, hi);
      load_rows<T, DP>(kf, (const T*)p.k + w.row0 * p.k_row + kv * p.k_head, k_at, p.dim, hi);
      load_rows<T, DP>(df, (const T*)p.dout + w.col0 * p.do_row + head * p.do_head, d_at, p.dim, hi);
      load_rows<T, DP>(vf, (const T*)p.v + w.row0 * p.v_row + kv * p.v_head, v_at, p.dim, hi);
    };
    load(h0);
    const int lane_of_item = lane;
    for (int head = h0; head < h0 + each; ++head) {
      const int lane = here(lane_of_item), col = lane & 31, hi = lane >> 5;
      const int kv = SHARE ? uniform(head / share) : head;
      keep_rows<T, DP>(qf, p.dim, hi, live);
      keep_rows<T, DP>(kf, p.dim, hi, key);
      keep_rows<T, DP>(df, p.dim, hi, live);
      keep_rows<T, DP>(vf, p.dim, hi, key);
      f32x16 acc = acc_zero(), dp = acc_zero();
#pragma unroll
      for (int c = 0; c < DP / 16; ++c)
        if (c * 16 < p.dim) {
          acc = Mma<T>::run(kf[c], qf[c], acc);
          dp = Mma<T>::run(vf[c], df[c], dp);
        }
      tile_sync<false>();
      put_rows<T, DP>(lds.dout, df, col, hi);
      put_rows<T, DP>(lds.q, qf, col, hi);
      put_rows<T, DP>(lds.k, kf, col, hi);
      if (head + 1 < h0 + each) load(head + 1);  // in flight while this head is computed
      const float slope = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, slopes[head])));
      float s[16], t[16];
      small_scores<T>(p, g, acc, scale, slope * kLog2e, tab + head * n_rel, live ? nk : 0, hi, s);
      small_exp<T>(s);
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
        sum = wave_sum(sum);
        if (lane == head) dslope += sum;
      }
      if (p.part_hist) {
        float run = 0.f;
        g.here();
#pragma unroll
        for (int r = 0; r < 16; ++r) {  // (runs of keys of one residue are added up in the lane first)
          run += t[r];
          if (r == 15 || g.at(r < 15 ? r + 1 : 15) != g.at(r)) {
            __hip_atomic_fetch_add(lds.hist + head * n_rel + g.at(r), run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
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
      WeightTile<T>::put(lds.score, split8<T>(s), split8<T>(s + 8), col, hi);
      tile_sync<false>();
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
        if (d * 32 < p.dim) {
          if (!SHARE) dv[d] = acc_zero();
          dv[d] = mma<T>(load_t<T, DP>(lds.dout, 0, d * 32, lane, hi), WeightTile<T>::get(lds.score, 0, lane, hi), dv[d]);
          if (nq > 16)  // (the other half of the contraction is all zeros)
            dv[d] = mma<T>(load_t<T, DP>(lds.dout, 1, d * 32, lane, hi), WeightTile<T>::get(lds.score, 1, lane, hi), dv[d]);
        }
      tile_sync<false>();
      const Weights<T> t0 = split8<T>(t), t1 = split8<T>(t + 8);
      WeightTile<T>::put(lds.score, t0, t1, col, hi);
      tile_sync<false>();
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        if (d * 32 >= p.dim) continue;
        f32x16 x = acc_zero();
        x = mma<T>(load_t<T, DP>(lds.q, 0, d * 32, lane, hi), WeightTile<T>::get(lds.score, 0, lane, hi), x);
        if (nq > 16) x = mma<T>(load_t<T, DP>(lds.q, 1, d * 32, lane, hi), WeightTile<T>::get(lds.score, 1, lane, hi), x);
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] = SHARE ? dk[d][r] + x[r] * down : x[r] * down;
      }
      const float f = p.scale * down;
      T* oq = (T*)p.dq + ((int64_t)w.col0 * p.heads + head) * p.dim;
      const uint32_t oq_at = (uint32_t)(col * p.heads) * p.dim;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        if (d * 32 >= p.dim) continue;
        f32x16 x = acc_zero();
        x = mma<T>(load_t<T, DP>(lds.k, 0, d * 32, lane, hi), t0, x);
        if (nk > 16) x = mma<T>(load_t<T, DP>(lds.k, 1, d * 32, lane, hi), t1, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = d * 32 + 8 * k + 4 * hi;
          if (live && e < p.dim) store4<T>(oq + (oq_at + e), x[4 * k] * f, x[4 * k + 1] * f, x[4 * k + 2] * f, x[4 * k + 3] * f);
        }
      }
      if (!SHARE || head % share == share - 1) {
        constexpr float PDOWN = 1.f / PUP;
        T* ok = (T*)p.dk + ((int64_t)w.row0 * p.kv_heads + kv) * p.dim;
        T* ov = (T*)p.dv + ((int64_t)w.row0 * p.kv_heads + kv) * p.dim;
        const uint32_t ok_at = (uint32_t)(col * p.kv_heads) * p.dim;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int e = d * 32 + 8 * k + 4 * hi;
            if (!key || e >= p.dim) continue;
            store4<T>(ok + (ok_at + e), dk[d][4 * k] * p.scale, dk[d][4 * k + 1] * p.scale, dk[d][4 * k + 2] * p.scale, dk[d][4 * k + 3] * p.scale);
            store4<T>(ov + (ok_at + e), dv[d][4 * k] * PDOWN, dv[d][4 * k + 1] * PDOWN, dv[d][4 * k + 2] * PDOWN, dv[d][4 * k + 3] * PDOWN);
          }
          if (SHARE) dk[d] = acc_zero(), dv[d] = acc_zero();
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
        const float dx = q.x - k.x, dy = q.y - k.y, dz = q.z - k.z;
        const float f = live ? weight[r] * inverse_dist(g.far[r]) : 0.f;
        x -= f * dx, y -= f * dy, z -= f * dz;
        lds.pull[col * kPullLd + row] = f;
      }
      tile_sync<false>();
      const float4 k = lds.kpos[col];
      float u = 0.f, v = 0.f, t = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = acc_row(r, hi);  // (rows beyond the last query pull by 0)
        const float4 o = lds.qpos[row];
        const float f = lds.pull[row * kPullLd + col];
        u += f * (o.x - k.x), v += f * (o.y - k.y), t += f * (o.z - k.z);
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
  const int lane = lane_of_wave;
  const int64_t part = p.part0 + worker;
  for (int head = h0; head < h0 + each; ++head) {
    if (p.part_slope) {
      const float sum = __shfl(dslope, head, 64);
      if (lane < kCoopWaves) p.part_slope[(head * (int64_t)p.parts + part) * kCoopWaves + lane] = lane ? 0.f : sum;
    }
    if (p.part_hist)
      for (int i = lane; i < n_rel; i += 64) p.part_hist[((int64_t)head * n_rel + i) * p.parts + part] = lds.hist[head * n_rel + i];
  }
}

// ---- fragments of two tiles: up to 64 queries and 64 keys ----
// A wave takes a fragment and one key head.  All keys of a query are in registers (two tiles side by side), so here too
// every score is computed once: 4 tiles instead of the 12 that the passes of attention_bwd.hip visit.  492 of 4096 fragments
// (33 ... 44 rows), 8 heads: f32 126 us (the three passes 63 more), bf16 105 us (47 more).  Bound by latency: 16-bit rows spill
// at two waves per SIMD and still beat one wave (all fragments, both directions, 323 and 345 us); float32 rows do not (430 us
// at two, 407 at one).
template <typename T, int DP>
struct PairLds {
  static constexpr size_t A = TileShape<T, DP>::BYTES, B = WeightTile<T>::BYTES;
  static constexpr size_t PULL = sizeof(float) * kTile * kPullLd;
  static constexpr size_t S = B > PULL ? B : PULL;
  T *k, *q, *dout, *score;  // k: two tiles; score: P, dS, and the pulls of one tile
  float* pull;
  float4 *kpos, *qpos;      // [64]
  int *kres, *qres;
  float *tab, *hist;
  __device__ __forceinline__ PairLds(char* p, int n_rel) {
    k = (T*)p;
    q = (T*)(p + 2 * A);
    dout = (T*)(p + 3 * A);
    score = (T*)(p + 4 * A);
    pull = (float*)(p + 4 * A);
    kpos = (float4*)(p + ((4 * A + S + 15) & ~(size_t)15));
    qpos = kpos + 2 * kTile;
    kres = (int*)(qpos + 2 * kTile);
    qres = kres + 2 * kTile;
    tab = (float*)(qres + 2 * kTile);
    hist = tab + n_rel;
  }
  static size_t bytes(int n_rel) {
    return (((4 * A + S + 15) & ~(size_t)15) + 4 * kTile * (sizeof(float4) + sizeof(int)) + 2 * sizeof(float) * n_rel + 15) & ~(size_t)15;
  }
};

template <typename T, int DP>
__global__ __launch_bounds__(256, (sizeof(T) == 4 ? 1 : 2)) void k_attn_pair_bwd(AttnParams p, size_t per_wave) {
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  constexpr bool HALF = is_half<T>();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane_of_wave = threadIdx.x & 63;
  const uint32_t id = blockIdx.x * (blockDim.x >> 6) + wave;
  if (id >= (uint32_t)p.workers * p.heads) return;
  const int head = uniform(id % p.heads), worker = uniform(id / p.heads);  // (key heads are not shared: heads == kv_heads)
  const int n_rel = p.table ? p.n_rel : 0;
  const PairLds<T, DP> lds(lds_raw + wave * per_wave, n_rel);
  if (p.table) expand_table(lds.tab, p.table + (int64_t)head * p.n_buckets, p.lut, n_rel, lane_of_wave, 64);
  for (int i = lane_of_wave; i < n_rel; i += 64) lds.hist[i] = 0.f;
  const float scale = p.scale * kLog2e, slope = p.slope ? p.slope[head] : 0.f, slope2 = slope * kLog2e;
  constexpr float PUP = HALF ? 0x1p14f : 1.f;
  float dslope = 0.f;

  for (int item = worker; item < p.count; item += p.workers) {
    const AttnWork w = load_work(p.work, item);
    const int nq = w.cols, nk = w.row1 - w.row0;
    const int lane = here(lane_of_wave), col = lane & 31, hi = lane >> 5;
    tile_sync<false>();
    {
      const int64_t kr = (int64_t)w.row0 + (lane < nk ? lane : 0), qr = (int64_t)w.col0 + (lane < nq ? lane : 0);
      if (p.slope) {
        lds.kpos[lane] = make_float4(p.k_pos[3 * kr], p.k_pos[3 * kr + 1], p.k_pos[3 * kr + 2], 0.f);
        lds.qpos[lane] = make_float4(p.q_pos[3 * qr], p.q_pos[3 * qr + 1], p.q_pos[3 * qr + 2], 0.f);
      }
      if (p.table) lds.kres[lane] = p.k_res[kr], lds.qres[lane] = p.q_res[qr];
    }
    typename vec8<T>::type vf[2][DP / 16];
    const T* kb = (const T*)p.k + w.row0 * p.k_row + head * p.k_head;
    const T* vb = (const T*)p.v + w.row0 * p.v_row + head * p.v_head;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int key = j * kTile + col;
      typename vec8<T>::type kf[DP / 16];
      load_rows<T, DP>(kf, kb, (key < nk ? key : 0) * (uint32_t)p.k_row, p.dim, hi);
      load_rows<T, DP>(vf[j], vb, (key < nk ? key : 0) * (uint32_t)p.v_row, p.dim, hi);
      keep_rows<T, DP>(kf, p.dim, hi, key < nk);
      keep_rows<T, DP>(vf[j], p.dim, hi, key < nk);
      put_rows<T, DP>(lds.k + j * kTile * TileShape<T, DP>::LD, kf, col, hi);
    }
    f32x16 dk[2][DP / 32], dv[2][DP / 32];
    float gk[2][3];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      gk[j][0] = gk[j][1] = gk[j][2] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) dk[j][d] = acc_zero(), dv[j][d] = acc_zero();
    }
    const int lane_of_item = lane;

    for (int i0 = 0; i0 < nq; i0 += kTile) {
      const int lane = here(lane_of_item), col = lane & 31, hi = lane >> 5;
      const bool live = i0 + col < nq;
      const int n_i = nq - i0 < kTile ? nq - i0 : kTile;
      const int64_t q_row = (int64_t)w.col0 + i0 + (live ? col : 0);
      const uint32_t in = live ? i0 + col : 0;
      typename vec8<T>::type qf[DP / 16], df[DP / 16];
      load_rows<T, DP>(qf, (const T*)p.q + w.col0 * p.q_row + head * p.q_head, in * (uint32_t)p.q_row, p.dim, hi);
      load_rows<T, DP>(df, (const T*)p.dout + w.col0 * p.do_row + head * p.do_head, in * (uint32_t)p.do_row, p.dim, hi);
      keep_rows<T, DP>(qf, p.dim, hi, live);
      keep_rows<T, DP>(df, p.dim, hi, live);
      tile_sync<false>();
      put_rows<T, DP>(lds.q, qf, col, hi);
      put_rows<T, DP>(lds.dout, df, col, hi);
      tile_sync<false>();

      float s[2][16], t[2][16];
      const float4 q = lds.qpos[i0 + col];
      const int res = p.table ? lds.qres[i0 + col] : 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const T* kt = lds.k + j * kTile * TileShape<T, DP>::LD;
        f32x16 acc = acc_zero(), dp = acc_zero();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
          if (c * 16 < p.dim) {
            acc = Mma<T>::run(load_n<T, DP>(kt, c, col, hi), qf[c], acc);
            dp = Mma<T>::run(vf[j][c], df[c], dp);
          }
        int limit = live ? nk - j * kTile : 0;
        compute_here(limit);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] = acc[r] * scale, t[j][r] = dp[r];
        if (p.slope) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float4 k = lds.kpos[j * kTile + acc_row(r, hi)];
            s[j][r] -= slope2 * pair_dist(q.x - k.x, q.y - k.y, q.z - k.z);
          }
        }
        if (p.table) {
          float b[16];
#pragma unroll
          for (int r = 0; r < 16; ++r) b[r] = lds.tab[rel_index(lds.kres[j * kTile + acc_row(r, hi)], res, p.reach)];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[j][r] += b[r];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] = acc_row(r, hi) < limit ? s[j][r] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fmaxf(s[0][r], s[1][r]));
      top = fmaxf(top, other_half(top));
      const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] = __builtin_amdgcn_exp2f(s[j][r] - ref);
      float l = tile_sum(s[0]) + tile_sum(s[1]), delta;
      {
        float u[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) u[r] = s[0][r] * t[0][r] + s[1][r] * t[1][r];
        delta = tile_sum(u);
      }
      l += other_half(l);
      delta += other_half(delta);
      const float inv_l = l == 0.f ? 0.f : 1.f / l;
      delta *= inv_l;
      float gx = 0.f, gy = 0.f, gz = 0.f, largest = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[j][r] *= inv_l;                        // P
          t[j][r] = s[j][r] * (t[j][r] - delta);  // dS
          if (HALF) largest = fmaxf(largest, fabsf(t[j][r]));
        }
      float up = 1.f, down = 1.f;
      if constexpr (HALF) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor(largest, o, 64));
        if (largest >= 0x1p-80f && largest < INFINITY) {
          up = ldexpf(1.f, 14 - ilogbf(largest));
          down = ldexpf(1.f, ilogbf(largest) - 14);
        }
      }
      f32x16 dq[DP / 32];
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) dq[d] = acc_zero();
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n_j = nk - j * kTile;  // (the second tile may be empty: all its terms are 0)
        const T* kt = lds.k + j * kTile * TileShape<T, DP>::LD;
        if (n_j <= 0) continue;
        if (p.part_hist) {
          float run = 0.f;
          int at = rel_index(lds.kres[j * kTile + acc_row(0, hi)], res, p.reach);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            run += t[j][r];
            const int then = r < 15 ? rel_index(lds.kres[j * kTile + acc_row(r < 15 ? r + 1 : 15, hi)], res, p.reach) : -1;
            if (then != at) {
              __hip_atomic_fetch_add(lds.hist + at, run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
              run = 0.f;
            }
            at = then;
          }
        }
        if (p.slope) {
          tile_sync<false>();
          float sum = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float4 k = lds.kpos[j * kTile + acc_row(r, hi)];
            const float dx = q.x - k.x, dy = q.y - k.y, dz = q.z - k.z;
            const float far = pair_dist(dx, dy, dz);
            sum -= t[j][r] * far;
            const float f = live ? slope * t[j][r] * inverse_dist(far) : 0.f;
            gx -= f * dx, gy -= f * dy, gz -= f * dz;
            if (p.dpos) lds.pull[col * kPullLd + acc_row(r, hi)] = f;
          }
          dslope += sum;
          tile_sync<false>();
          if (p.dpos) {
            const float4 k = lds.kpos[j * kTile + col];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              // rows beyond the last query pull by 0; 16-bit rows skip them, which keeps the loads from being hoisted into
              // registers that spill (bf16, all fragments, both directions: 347 us without the branch, 323 us with it)
              const int row = acc_row(r, hi);
              if (sizeof(T) == 4 || row < n_i) {
                const float4 o = lds.qpos[i0 + row];
                const float f = lds.pull[row * kPullLd + col];
                gk[j][0] += f * (o.x - k.x), gk[j][1] += f * (o.y - k.y), gk[j][2] += f * (o.z - k.z);
              }
            }
          }
        }
        float u[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[j][r] *= PUP, u[r] = t[j][r] * up;
        tile_sync<false>();
        WeightTile<T>::put(lds.score, split8<T>(s[j]), split8<T>(s[j] + 8), col, hi);
        tile_sync<false>();
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
          if (d * 32 < p.dim) {
            dv[j][d] = mma<T>(load_t<T, DP>(lds.dout, 0, d * 32, lane, hi), WeightTile<T>::get(lds.score, 0, lane, hi), dv[j][d]);
            if (n_i > 16)
              dv[j][d] = mma<T>(load_t<T, DP>(lds.dout, 1, d * 32, lane, hi), WeightTile<T>::get(lds.score, 1, lane, hi), dv[j][d]);
          }
        tile_sync<false>();
        const Weights<T> u0 = split8<T>(u), u1 = split8<T>(u + 8);
        WeightTile<T>::put(lds.score, u0, u1, col, hi);
        tile_sync<false>();
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) {
          if (d * 32 >= p.dim) continue;
          f32x16 x = acc_zero();
          x = mma<T>(load_t<T, DP>(lds.q, 0, d * 32, lane, hi), WeightTile<T>::get(lds.score, 0, lane, hi), x);
          if (n_i > 16) x = mma<T>(load_t<T, DP>(lds.q, 1, d * 32, lane, hi), WeightTile<T>::get(lds.score, 1, lane, hi), x);
#pragma unroll
          for (int r = 0; r < 16; ++r) dk[j][d][r] += x[r] * down;
          dq[d] = mma<T>(load_t<T, DP>(kt, 0, d * 32, lane, hi), u0, dq[d]);
          if (n_j > 16) dq[d] = mma<T>(load_t<T, DP>(kt, 1, d * 32, lane, hi), u1, dq[d]);
        }
      }
      if (live) store_column<T, DP>((T*)p.dq + (q_row * p.heads + head) * p.dim, dq, p.scale * down, p.dim, hi);
      if (p.dpos) {
        gx += other_half(gx), gy += other_half(gy), gz += other_half(gz);
        float* g = p.part_pos_q + (head * p.rows_q + q_row) * 3;
        if (live && hi == 0) g[0] = gx, g[1] = gy, g[2] = gz;
      }
    }

#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const bool key = j * kTile + col < nk;
      const int64_t k_row = (int64_t)w.row0 + (key ? j * kTile + col : 0);
      if (key) {
        store_column<T, DP>((T*)p.dk + (k_row * p.heads + head) * p.dim, dk[j], p.scale, p.dim, hi);
        store_column<T, DP>((T*)p.dv + (k_row * p.heads + head) * p.dim, dv[j], 1.f / PUP, p.dim, hi);
      }
      if (p.dpos) {
        const float x = gk[j][0] + other_half(gk[j][0]), y = gk[j][1] + other_half(gk[j][1]), z = gk[j][2] + other_half(gk[j][2]);
        float* g = p.part_pos_k + (head * p.rows_k + k_row) * 3;
        if (key && hi == 0) g[0] = x, g[1] = y, g[2] = z;
      }
    }
  }

  tile_sync<false>();
  const int64_t part = p.part0 + worker;
  if (p.part_slope) {
    const float sum = wave_sum(dslope);
    if (lane_of_wave < kCoopWaves) p.part_slope[(head * (int64_t)p.parts + part) * kCoopWaves + lane_of_wave] = lane_of_wave ? 0.f : sum;
  }
  if (p.part_hist)
    for (int i = lane_of_wave; i < n_rel; i += 64) p.part_hist[((int64_t)head * n_rel + i) * p.parts + part] = lds.hist[i];
}

template <typename T, int DP>
static int pair_launch(const AttnParams& p, hipStream_t st) {
  const size_t bytes = PairLds<T, DP>::bytes(p.table ? p.n_rel : 0);
  const int64_t total = (int64_t)p.workers * p.heads;
  const int waves = lone_waves(bytes);
  if (!allow_lds((const void*)k_attn_pair_bwd<T, DP>, waves * bytes)) return -5;
  hipLaunchKernelGGL((k_attn_pair_bwd<T, DP>), dim3((unsigned)((total + waves - 1) / waves)), dim3(64 * waves),
                     waves * bytes, st, p, bytes);
  return 0;
}

int attn_pair_backward(int dtype, const AttnParams& p, hipStream_t st) {
  switch (dtype) {
    case VSN_F32: return p.dim <= 32 ? pair_launch<float, 32>(p, st) : pair_launch<float, 64>(p, st);
    case VSN_BF16: return p.dim <= 32 ? pair_launch<__bf16, 32>(p, st) : pair_launch<__bf16, 64>(p, st);
    default: return p.dim <= 32 ? pair_launch<_Float16, 32>(p, st) : pair_launch<_Float16, 64>(p, st);
  }
}

template <typename T, int DP>
static int small_launch(AttnParams p, int groups, bool backward, hipStream_t st) {
  const int n_rel = p.table ? p.n_rel : 0;
  const size_t tab = (sizeof(float) * p.heads * (n_rel + 1) + 15) & ~(size_t)15;
  const size_t bytes = SmallLds<T, DP>::bytes(p.heads, n_rel, backward);
  const int64_t total = (int64_t)(backward ? p.workers : p.count) * groups;
  int waves = total <= 1024 ? 1 : 4;
  while (waves > 1 && tab + waves * bytes > kLdsPerCu / 2) waves /= 2;
  const size_t lds = tab + waves * bytes;
  const dim3 grid((unsigned)((total + waves - 1) / waves)), block(64 * waves);
  if (backward) {
    if (p.heads == p.kv_heads) {
      if (!allow_lds((const void*)k_attn_small_bwd<T, DP, false>, lds)) return -5;
      hipLaunchKernelGGL((k_attn_small_bwd<T, DP, false>), grid, block, lds, st, p, bytes, groups);
    } else {
      if (!allow_lds((const void*)k_attn_small_bwd<T, DP, true>, lds)) return -5;
      hipLaunchKernelGGL((k_attn_small_bwd<T, DP, true>), grid, block, lds, st, p, bytes, groups);
    }
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
