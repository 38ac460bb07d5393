// Fragment attention: what the forward and the backward kernels share.
//
// For a query row i and a key row j of one fragment, head a (key head a / group):
//   s_ij = scale q_i.k_j - slope_a |x_i - x_j| + table[a][bucket(res_j - res_i)],   P = softmax_j(s),   o_i = sum_j P_ij v_j
//
// A wave works on tiles of 32 x 32 scores in the registers of one 32x32 MFMA accumulator: lane = column (lane & 31), the
// 16 registers = rows acc_row(r).  The tile is computed with the rows' operand from LDS and the columns' operand from
// registers, so everything that belongs to a column (running maximum and sum, position, residue, gradient scale) is the
// lane's own, and a column of P or dS is already the B operand of the next product: that product contracts over the
// tile's rows, whose order inside a contraction is free, and takes its A operand in the same order (load_t).
// float16 exponentials go up to 2^14 (their reference is the maximum minus 14): at 1, what lies under 2^-25 of the largest
// term would be lost to the product and counted in the sum, 3 % of a row of 10^6 keys.
// Float32 runs the same tiles on the float32 matrix instruction (8 of 2 rows instead of one of 16), each tile's product
// in an accumulator of its own that is then added to the sum: a chain of one addition per two rows would lose half of a
// decimal digit over a protein of some thousand atoms.
// Scores are in units of log 2 (scale, slopes and table are multiplied by log2 e beforehand), so the exponential needs no
// product of its own, and no rounding of one.
#pragma once
#include "typed.h"

namespace vsn {

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kTile = 32;         // rows and columns of a tile
constexpr int kCoopWaves = 4;     // waves that share the tiles of one workgroup (128 columns of one head)
constexpr int kMaxReach = 1023;   // clipped residue difference: 2 reach + 1 table entries in LDS

// One block of columns (queries in the forward and dq passes, keys in the dk / dv pass) against a run of rows.
struct AttnWork {
  int col0, cols;  // first column row, number of columns (<= 32, or <= 128 where the workgroup shares tiles)
  int row0, row1;  // the rows it meets
  int slot;        // >= 0: one of several pieces of a run of rows; its partial results go to slots slot + wave
  int slot0, slots, step;  // the pieces' slots: slot0 + wave + i step, i < slots
};
// Partial results to join: `cols` (<= 32) columns from col0, slots slot0 + i step, i < slots
struct AttnJoin {
  int col0, cols, slot0, slots, step;
};

struct AttnParams {
  const AttnWork* work;
  int count;              // work items
  int workers, part0;     // backward: workers per head of this launch, first partial sum of this launch
  int parts;              // partial sums per head over all launches
  int heads, kv_heads, dim;
  int reach, n_rel, n_buckets;
  const int* lut;         // [n_rel] bucket of a clipped difference
  const void *q, *k, *v, *dout;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;
  const float *q_pos, *k_pos, *slope;
  const int *q_res, *k_res;
  const float* table;     // [heads][n_buckets]
  float scale;
  int64_t rows_q, rows_k; // rows of the arrays (statistics and partial sums are laid out by them)
  void* out;
  int64_t out_row, out_head;
  float2* stats;          // [heads][rows_q] {maximum in units of log 2, sum of exponentials}
  // pieces of split runs
  float *part_o, *part_o2;  // [slot][heads][32][dim]: unnormalised output; dq; dk and dv
  float2* part_ml;          // [slot][heads][32]: maximum and sum; sums of e and of e dP
  float* part_g;            // [slot][heads][32][4]: a column's positions' gradient
  const AttnJoin* join;
  // backward
  float2* delta;          // [heads][rows_q] {D, 1 / sum of exponentials}
  void *dq, *dk, *dv;     // contiguous
  float* part_pos_q;      // [heads][rows_q][3] or null
  float* part_pos_k;      // [kv_heads][rows_k][3] or null
  float* part_slope;      // [heads][4 parts] or null
  float* part_hist;       // [heads][n_rel][parts] or null
  float *dpos, *dq_pos, *dslope, *dtable;
};

// A value that is the same for all lanes, in a scalar register (an integer division leaves it in a vector register, and
// with it every address computed from it).
__device__ __forceinline__ int uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane((int)v); }
// Keeps what is computed from `v` inside the loop that uses it.  The compiler otherwise holds every address and comparison
// that does not change over the loop in a register of its own: a hundred of them, which is a wave or two per SIMD.
template <typename V>
__device__ __forceinline__ void compute_here(V& v) {
  asm volatile("" : "+v"(v));
}
__device__ __forceinline__ int here(int v) {
  compute_here(v);
  return v;
}

// A work item in scalar registers: it is the same for all lanes, which the compiler cannot know of a value that it has to
// load behind the stores of the item before.
__device__ __forceinline__ AttnWork load_work(const AttnWork* work, int64_t at) {
  AttnWork w = work[at];
  w.col0 = __builtin_amdgcn_readfirstlane(w.col0), w.cols = __builtin_amdgcn_readfirstlane(w.cols);
  w.row0 = __builtin_amdgcn_readfirstlane(w.row0), w.row1 = __builtin_amdgcn_readfirstlane(w.row1);
  w.slot = __builtin_amdgcn_readfirstlane(w.slot), w.slot0 = __builtin_amdgcn_readfirstlane(w.slot0);
  w.slots = __builtin_amdgcn_readfirstlane(w.slots), w.step = __builtin_amdgcn_readfirstlane(w.step);
  return w;
}

template <typename T>
constexpr bool is_half() {
  return __is_same(T, _Float16);
}
// The reference that a maximum stands for in the exponentials.  (From 2^25 on float32 could round the difference of 14 to 16,
// and 2^16 is no float16 any more; below 2^24, where scores still tell one unit from the next, it is at most 15.)
constexpr float kExact = 0x1p24f;
template <typename T>
__device__ __forceinline__ float exp_ref(float top) {
  return is_half<T>() && fabsf(top) < kExact ? top - 14.f : top;
}
// what a caller keeps: the maximum, and the sum of the exponentials relative to it
template <typename T>
__device__ __forceinline__ float2 attn_stats(float ref, float sum) {
  return is_half<T>() && fabsf(ref + 14.f) < kExact ? make_float2(ref + 14.f, sum * 0x1p-14f) : make_float2(ref, sum);
}

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
  static __device__ __forceinline__ f32x16 run(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<_Float16> {
  static __device__ __forceinline__ f32x16 run(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> {
  static __device__ __forceinline__ f32x16 run(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int t = 0; t < 8; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
    return c;
  }
};

// row of accumulator register r in the lane's half
__device__ __forceinline__ int acc_row(int r, int hi) { return 8 * (r >> 2) + 4 * hi + (r & 3); }

__device__ __forceinline__ f32x16 acc_zero() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

template <typename T, int DP>
struct TileShape {
  static constexpr int LD = DP + 16 / (int)sizeof(T);            // 16 bytes of padding per row: 16-byte reads of 8 rows
                                                                 // in a row fall on different banks
  static constexpr int EPC = 16 / (int)sizeof(T);                // elements per 16-byte chunk
  static constexpr int CPR = DP / EPC;                           // chunks per row
  static constexpr int CHUNKS = kTile * CPR;                     // chunks per tile
  static constexpr size_t BYTES = sizeof(T) * kTile * LD;
};

// Copies two tiles (32 rows of two arrays) into LDS by way of registers, so the loads of the next tiles can be in flight
// while the present ones are computed with.  Rows and columns beyond the end are zeros.
template <typename T, int DP, int THREADS>
struct TilePair {
  typedef TileShape<T, DP> S;
  static constexpr int N = (2 * S::CHUNKS + THREADS - 1) / THREADS;
  uint4 reg[N];
  __device__ __forceinline__ void load(const T* a, int64_t a_row, const T* b, int64_t b_row, int rows, int dim, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * THREADS;
      const bool second = c >= S::CHUNKS;
      const int rest = c >= 2 * S::CHUNKS ? 0 : second ? c - S::CHUNKS : c;
      const int row = rest / S::CPR, at = rest % S::CPR * S::EPC;
      // (loads without a branch, from a row and a column that are there; what is beyond the end is zeroed on the way to LDS)
      const int r = row < rows ? row : 0, e = at < dim ? at : 0;
      reg[i] = *(const uint4*)((second ? b + r * b_row : a + r * a_row) + e);
    }
  }
  __device__ __forceinline__ void store(T* a, T* b, int rows, int dim, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * THREADS;
      if (c < 2 * S::CHUNKS) {
        const int rest = c >= S::CHUNKS ? c - S::CHUNKS : c;
        const int row = rest / S::CPR, at = rest % S::CPR * S::EPC;
        *(uint4*)((c >= S::CHUNKS ? b : a) + row * S::LD + at) = row < rows && at < dim ? reg[i] : make_uint4(0, 0, 0, 0);
      }
    }
  }
};

// Orders LDS writes of some lanes before reads of others: a barrier where the workgroup shares the tiles, and an order
// for the compiler where they are the wave's own (a wave's LDS accesses are carried out in program order).
template <bool COOP>
__device__ __forceinline__ void tile_sync() {
  if constexpr (COOP) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// A operand "row of the tile": lane's row (lane & 31), elements c 16 + hi 8 ... + 7
template <typename T, int DP>
__device__ __forceinline__ typename vec8<T>::type load_n(const T* tile, int c, int col, int hi) {
  return *(const typename vec8<T>::type*)(tile + col * TileShape<T, DP>::LD + c * 16 + hi * 8);
}

// A operand "column of the tile": lane's column d0 + (lane & 31), rows acc_row(8 c + 0 ... 7) - the order in which a lane
// holds its scores.  16-bit types: two transposing LDS reads of 4 rows x 16 columns per 16 lanes (lane 4 e + j / 4 of a
// group supplies row e, four columns from 4 (j & 3); lane j receives column j).
template <typename T, int DP>
__device__ __forceinline__ typename vec8<T>::type load_t(const T* tile, int c, int d0, int lane, int hi) {
  typename vec8<T>::type f;
  constexpr int LD = TileShape<T, DP>::LD;
  if constexpr (sizeof(T) == 4) {
    const float* p = tile + d0 + (lane & 31);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[acc_row(8 * c + i, hi) * LD];
  } else {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int j = lane & 15;
    const T* p = tile + (16 * c + 4 * hi + (j >> 2)) * LD + d0 + (lane & 16) + 4 * (j & 3);
    s16x4 part[2];
    part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * LD));
    __builtin_memcpy(&f, part, 16);
  }
  return f;
}

// eight elements of a global row as a B operand (column operand), zeros beyond the end
template <typename T>
__device__ __forceinline__ typename vec8<T>::type load_col(const T* row, int at, int dim, bool live) {
  typename vec8<T>::type f;
  if (live && at < dim) {
    f = *(const typename vec8<T>::type*)(row + at);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (T)0.f;
  }
  return f;
}

// Eight weights (P, dS) as B operands of a product.  16-bit rows take them in two parts, hi + lo: one rounding to the rows'
// type would put an error as large as the result's own rounding into every term, which the caller of 16-bit rows did not
// ask for; two leave 2^-18 (bf16) and 2^-24 (f16) of a term.  The second product costs little, as the matrix units wait for
// the vector ones; what it costs is the split, 7 instructions per pair of weights (bf16).  17 882 atoms bf16, dim 32: forward
// 1.35 -> 1.62 ms, both directions 9.2 -> 10.2 ms; 6007 atoms f16, dim 64, both 1.48 -> 1.65 ms; fragments gain nothing by
// less (4096 of them bf16, both 0.332 and 0.338 ms).
template <typename T>
struct Weights {
  typename vec8<T>::type hi, lo;
};
template <>
struct Weights<float> {
  f32x8 hi;
};
template <typename T>
__device__ __forceinline__ Weights<T> split8(const float* p) {
  Weights<T> w;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w.hi[i] = (T)p[i];
    if constexpr (sizeof(T) == 2) w.lo[i] = (T)(p[i] - (float)w.hi[i]);
  }
  return w;
}
template <typename T>
__device__ __forceinline__ f32x16 mma(typename vec8<T>::type a, const Weights<T>& b, f32x16 c) {
  c = Mma<T>::run(a, b.hi, c);
  if constexpr (sizeof(T) == 2) c = Mma<T>::run(a, b.lo, c);
  return c;
}

// four consecutive elements of an output row
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
  T v[4] = {(T)a, (T)b, (T)c, (T)d};
  if constexpr (sizeof(T) == 4)
    *(float4*)p = *(float4*)v;
  else
    *(uint2*)p = *(uint2*)v;
}

// a column of an accumulator as a row of an output
template <typename O, int DP>
__device__ __forceinline__ void store_column(O* o, const f32x16 (&c)[DP / 32], float f, int dim, int hi) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int e = d * 32 + 8 * g + 4 * hi;
      if (e < dim) store4<O>(o + e, c[d][4 * g] * f, c[d][4 * g + 1] * f, c[d][4 * g + 2] * f, c[d][4 * g + 3] * f);
    }
}

// |a - b| from the difference's components (the root instruction, off by at most one step), and its reciprocal: a huge
// finite number where the points coincide, where the difference itself and with it the direction is 0.
__device__ __forceinline__ float pair_dist(float dx, float dy, float dz) {
  return __builtin_amdgcn_sqrtf(dx * dx + dy * dy + dz * dz);
}
__device__ __forceinline__ float inverse_dist(float far) { return __builtin_amdgcn_rcpf(fmaxf(far, 1e-18f)); }

// index of the clipped difference of two residue numbers; the difference saturates
__device__ __forceinline__ int rel_index(int key_res, int query_res, int reach) {
  const int d = __builtin_elementwise_sub_sat(key_res, query_res);
  return __builtin_elementwise_min(__builtin_elementwise_max(d, -reach), reach) + reach;
}

// a table entry in units of log 2; the lowest float32 stays a finite value (a mask of it must not turn into -inf)
__device__ __forceinline__ float table_log2(float t) {
  const float v = t * kLog2e;
  return fabsf(t) < INFINITY ? __builtin_amdgcn_fmed3f(v, -3.4028235e38f, 3.4028235e38f) : v;
}

// This head's table by clipped difference, in LDS.  Loads go out eight at a time: one after the other, two dependent
// loads per 64 entries cost a wave of a 257-entry table more than its tiles.
__device__ __forceinline__ void expand_table(float* tab, const float* table, const int* lut, int n_rel, int tid,
                                             int threads) {
  for (int base = 0; base < n_rel; base += 8 * threads) {
    int at[8];
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = base + k * threads + tid;
      at[k] = lut[i < n_rel ? i : 0];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = table[at[k]];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = base + k * threads + tid;
      if (i < n_rel) tab[i] = table_log2(v[k]);
    }
  }
}

// c += a * b over one tile of 32 rows
template <typename T>
__device__ __forceinline__ void tile_mma(f32x16& c, typename vec8<T>::type a0, const Weights<T>& b0,
                                         typename vec8<T>::type a1, const Weights<T>& b1) {
  if constexpr (sizeof(T) == 4) {
    f32x16 t = mma<T>(a0, b0, acc_zero());
    t = mma<T>(a1, b1, t);
#pragma unroll
    for (int r = 0; r < 16; ++r) c[r] += t[r];
  } else {
    c = mma<T>(a0, b0, c);
    c = mma<T>(a1, b1, c);
  }
}

// Whether all differences of a tile are clipped to one end of the table: its index, or -1.  `row_res` is the residue of
// tile row (lane & 31), lo and hi the smallest and the largest residue of the wave's columns; sign +1: rows are keys.
__device__ __forceinline__ int clipped_end(int row_res, int lo, int hi, int sign, int reach) {
  const int up = sign > 0 ? __builtin_elementwise_sub_sat(row_res, hi) : __builtin_elementwise_sub_sat(lo, row_res);
  const int down = sign > 0 ? __builtin_elementwise_sub_sat(row_res, lo) : __builtin_elementwise_sub_sat(hi, row_res);
  return __all(up >= reach) ? 2 * reach : __all(down <= -reach) ? 0 : -1;
}
// smallest and largest of the wave's columns
__device__ __forceinline__ void column_range(int v, int& lo, int& hi) {
  lo = hi = v;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const int a = __shfl_xor(lo, o, 64), b = __shfl_xor(hi, o, 64);
    lo = a < lo ? a : lo, hi = b > hi ? b : hi;
  }
  lo = __builtin_amdgcn_readfirstlane(lo), hi = __builtin_amdgcn_readfirstlane(hi);
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// the 16 values of a tile's column half, added up pairwise
__device__ __forceinline__ float tile_sum(const float* v) {
  float t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = v[i] + v[i + 8];
  return ((t[0] + t[4]) + (t[2] + t[6])) + ((t[1] + t[5]) + (t[3] + t[7]));
}

// A sum over many tiles that carries its rounding error along (two-sum): sums over whole proteins whose terms cancel -
// sum_j dS_ij is 0 - keep the precision of their tiles.
struct LongSum {
  float s = 0.f, c = 0.f;
  __device__ __forceinline__ void add(float x) {
    const float t = s + x, b = t - s;
    c += (s - (t - b)) + (x - b);
    s = t;
  }
  __device__ __forceinline__ void scale(float f) { s *= f, c *= f; }
  __device__ __forceinline__ float both_halves() const {
    const float hi = s + other_half(s), lo = c + other_half(c);
    return hi + lo;
  }
  __device__ __forceinline__ float value() const { return s + c; }
};

// Waves per SIMD that the tile kernels are compiled for: as many as fit without spilling, left alone the compiler hoists
// its loads into twice the registers.  17 882 atoms bf16, dim 32, both directions at two, three and four: 11.5, 10.5 and 17.2 ms
// (the forward pass alone 1.7 ms at each); 6007 atoms f16, dim 64, at one and two: both directions 2.67 and 1.66 ms, forward
// 343 and 256 us.
template <typename T, int DP>
constexpr int forward_waves() {
  return DP <= 32 ? 3 : DP > 64 && sizeof(T) == 4 ? 1 : 2;
}
template <typename T, int DP>
constexpr int backward_waves() {
  return DP <= 32 && sizeof(T) == 2 ? 3 : DP <= 64 ? 2 : 1;
}

// wave-private (or shared) LDS of one work item
template <typename T, int DP>
struct AttnLds {
  static constexpr size_t TILES = 2 * TileShape<T, DP>::BYTES;
  static constexpr size_t META = kTile * (sizeof(float4) * 2 + sizeof(int));  // positions, statistics, residues
  T *a, *b;
  float4 *pos, *stat;
  int* res;
  float* tab;  // [n_rel] this head's table, expanded
  __device__ __forceinline__ explicit AttnLds(char* p) {
    a = (T*)p;
    b = (T*)(p + TileShape<T, DP>::BYTES);
    pos = (float4*)(p + TILES);
    stat = pos + kTile;
    res = (int*)(stat + kTile);
    tab = (float*)(res + kTile);
  }
  static size_t bytes(int n_rel) { return (TILES + META + sizeof(float) * n_rel + 15) & ~(size_t)15; }
};

}  // namespace vsn
