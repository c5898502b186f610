// Attention within a sliding window, with a few first keys that stay visible, forward and backward: fp32 arithmetic on
// the matrix cores (v_mfma_f32_16x16x4_f32), any head size up to 128, both storage types, any stride and alignment.
// The bf16 path for aligned heads is window_attn_mfma.hip.
//
//   S = scale Q K^T on visible pairs,  P = softmax(S),  O = P V;   with L = log-sum-exp of the rows of S:
//   P = exp(S - L),  dV = P^T dO,  dP = dO V^T,  dS = scale P (dP - rowsum(dO O)),  dQ = dS K,  dK = dS^T Q.
//
// A wave owns 16 rows (queries; keys in the dK / dV kernel) in registers and sweeps the other side in tiles of 64 rows
// held in LDS as fp32.  Products are D[rho][c] = sum_k X[rho][k] Y[c][k] with X from LDS and the wave's own rows Y on the
// lanes, so a softmax row is 16 registers and two exchanges, and the accumulators of the scores are the Y operand of the
// next product as they stand (k = 4 (lane / 16) + r, taken for r = 0 .. 3 in turn).  Scores never reach memory; tiles
// outside the window are never visited; dQ and dK / dV come from separate launches, so that no sum depends on the order
// of blocks.  Shared key heads: the dK / dV block walks the query heads of its group.
// 8192 tokens, 8 heads of 64, causal: 0.79 ms forward, 87 TFLOP/s of the 154 that a product of two 8192 x 8192 matrices
// reaches: the matrix unit (1/16 of bf16's rate) is busy 55 % of the launch, 2.5 waves a SIMD spend 64 % of their time waiting
// to issue and 19 % waiting for LDS or memory, and a CU is without waves for 12 %.  Where the blocks are few (16 packed texts
// of 100 - 1000 tokens, window 256: forward 82, dQ 108, dK and dV 155 us, 4.6 blocks of 5.5 tiles a CU in all) it is busy 31 -
// 35 %, with 1.6 waves.
#include "window_attn.h"
#include <algorithm>
#include <type_traits>

using namespace skwin;

namespace {

constexpr int NT = 64;     // rows per LDS tile
// Blocks per CU.  At width 128 the dK / dV kernel spills 23 registers for its second block and is faster for it (2 x 4096
// tokens, 8 heads, 2 key heads, window 512: 530 us alone, 428 by two; dQ 448 and 327).
constexpr int BLOCKS(int D) { return D <= 64 ? 3 : 2; }
constexpr int MAXD = 128;
constexpr int MAX_LEN = 1 << 29;   // positions, plus a window of both sequences' lengths, stay within 32 bits
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int MFMA_ROWS = 128;   // key rows of a block of the bf16 path

template <int D> struct Tile { float a[NT][D + 4]; };

__device__ __forceinline__ f32x4_t mfma4(float x, float y, f32x4_t acc) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, acc, 0, 0, 0);
}

// A tile of 64 rows on its way: loaded into registers while the tile before is multiplied, converted and written to LDS
// between two barriers.  Rows are clamped to the matrix; those whose bit in `ok` is clear, and columns beyond d, are
// written as zeros whatever they hold.
template <typename T> struct Load4;
template <> struct Load4<float> { typedef float4 raw; };
template <> struct Load4<bf16_t> { typedef uint2 raw; };
template <typename T, int D> struct Stage {
  typedef typename Load4<T>::raw raw;
  static constexpr int N = NT * (D / 4) / 256;
  raw r[N];
  __device__ __forceinline__ void load(const T* base, int64_t ld, int r0, int rows, int d, bool vec) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = threadIdx.x + 256 * k, row = e / (D / 4), c = (e - row * (D / 4)) * 4;
      const T* s = base + (int64_t)min(r0 + row, rows - 1) * ld;
      if (vec) {
        r[k] = *(const raw*)(s + (c < d ? c : 0));
      } else {
        T* w = (T*)&r[k];
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = s[c + x < d ? c + x : 0];
      }
    }
  }
  __device__ __forceinline__ void store(Tile<D>& t, uint64_t ok, int d) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int e = threadIdx.x + 256 * k, row = e / (D / 4), c = (e - row * (D / 4)) * 4;
      const T* w = (const T*)&r[k];
      const bool use = (ok >> row) & 1;
      float4 v;
      v.x = use && c < d ? Cvt<T>::to_f32(w[0]) : 0.f;
      v.y = use && c + 1 < d ? Cvt<T>::to_f32(w[1]) : 0.f;
      v.z = use && c + 2 < d ? Cvt<T>::to_f32(w[2]) : 0.f;
      v.w = use && c + 3 < d ? Cvt<T>::to_f32(w[3]) : 0.f;
      *(float4*)&t.a[row][c] = v;
    }
  }
};

// own row: y[s][j] = element 16 s + 4 g + j
template <typename T, int D>
__device__ __forceinline__ void load_own(f32x4_t (&y)[D / 16], const T* row, int d, int g, bool ok) {
#pragma unroll
  for (int s = 0; s < D / 16; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 16 * s + 4 * g + j;
      y[s][j] = ok && c < d ? Cvt<T>::to_f32(row[c]) : 0.f;
    }
}

// D[16 rows of the tile from row0][own] = sum over the head of tile x own
template <int D>
__device__ __forceinline__ f32x4_t dot_rows(const Tile<D>& t, int row0, const f32x4_t (&y)[D / 16], int lane) {
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const float4 x = *(const float4*)&t.a[row0 + (lane & 15)][16 * s + 4 * (lane >> 4)];
    acc = mfma4(x.x, y[s][0], acc);
    acc = mfma4(x.y, y[s][1], acc);
    acc = mfma4(x.z, y[s][2], acc);
    acc = mfma4(x.w, y[s][3], acc);
  }
  return acc;
}

// out[t][..] (columns 16 t + ..) += sum over tile rows row0 .. row0 + 15 of coef x tile
template <int D>
__device__ __forceinline__ void add_cols(f32x4_t (&out)[D / 16], const Tile<D>& t, int row0, const f32x4_t& coef, int lane) {
  const float* row = t.a[row0 + 4 * (lane >> 4)] + (lane & 15);
  // one row's columns on their way while the other's are multiplied (left to itself the compiler reads two, waits and
  // multiplies two: 4 x 4096 tokens, 8 heads of 64, window 1024: forward 404 -> 395 us; a single short text 28.5 -> 27.2)
  float x[2][D / 16];
#pragma unroll
  for (int c = 0; c < D / 16; ++c) x[0][c] = row[16 * c];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (r < 3) {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) x[(r + 1) & 1][c] = row[(r + 1) * (D + 4) + 16 * c];
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) out[c] = mfma4(x[r & 1][c], coef[r], out[c]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// own row's columns 16 t + 4 g + r
template <typename T, int D>
__device__ __forceinline__ void store_own(T* row, const f32x4_t (&o)[D / 16], float mul, int d, int g) {
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int c = 16 * t + 4 * g + r;
      if (c < d) row[c] = Cvt<T>::from_f32(o[t][r] * mul);
    }
}

// v where the lane's bit 16 k + r of a row mask (shifted right by 4 g) is set, else `other`
__device__ __forceinline__ float keep_or(float v, uint64_t mask, int k, int r, uint32_t other) {
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)(uint32_t)(mask >> (32 * (k >> 1))), 16 * (k & 1) + r, 1);
  return __uint_as_float((__float_as_uint(v) & m) | (other & ~m));
}

// Keys of a sequence as tiles: what forward and dQ sweep.
template <typename T, int D> struct KeySweep {
  const WinParams& p;
  const Seq& sq;
  const KeyTiles kt;
  const T *K, *V;
  const uint8_t* pad;
  Stage<T, D> k, v;
  int gone, beg, end;
  // the `cut`-th of `cuts` shares of the tiles that queries i0 .. i0 + 63 see
  __device__ __forceinline__ KeySweep(const WinParams& p_, const Seq& sq_, int b, int kh, int i0, int cut, int cuts)
      : p(p_), sq(sq_), kt(KeyTiles::of<NT>(p_, sq_, i0, min(i0 + 64, sq_.Lq))) {
    beg = (int)((int64_t)max(0, kt.n) * cut / cuts);
    end = (int)((int64_t)max(0, kt.n) * (cut + 1) / cuts);
    K = (const T*)p.K + sq.kbase * p.ldk + (int64_t)kh * p.d;
    V = (const T*)p.V + sq.kbase * p.ldv + (int64_t)kh * p.d;
    pad = p.key_pad ? p.key_pad + (int64_t)b * p.Lk : nullptr;
    gone = 0;
    if (beg < end) load(beg);
  }
  __device__ __forceinline__ int start(int t) const { return kt.start<NT>(t); }
  __device__ __forceinline__ int padding(int t) const { return pad ? pad[min(start(t) + (int)(threadIdx.x & 63), sq.Lk - 1)] : 0; }
  __device__ __forceinline__ uint64_t usable(int t, int no) const { return __ballot(kt.holds(start(t) + (int)(threadIdx.x & 63)) && !no); }
  __device__ __forceinline__ void load(int t) {
    const int j0 = start(t);
    gone = padding(t);
    k.load(K, p.ldk, j0, sq.Lk, p.d, p.vec);
    v.load(V, p.ldv, j0, sq.Lk, p.d, p.vec);
  }
  // tile t into LDS; the next one on its way.  Returns the keys that may be used.
  __device__ __forceinline__ uint64_t next(int t, Tile<D>& Ks, Tile<D>& Vs) {
    const uint64_t ok = usable(t, gone);
    __syncthreads();
    k.store(Ks, ok, p.d);
    v.store(Vs, ok, p.d);
    __syncthreads();
    if (t + 1 < end) load(t + 1);
    return ok;
  }
};

// whether any row of the wave has a bit among the 16 of piece k
__device__ __forceinline__ bool piece(uint64_t see, int k) { return __any(((see >> (16 * k)) & 0xffff) != 0); }

// ------------------------------------------------------------------------------ forward
template <typename T, int D>
__global__ __launch_bounds__(256, BLOCKS(D)) void window_fwd_kernel(WinParams p) {
  __shared__ __attribute__((aligned(16))) Tile<D> Ks;
  __shared__ __attribute__((aligned(16))) Tile<D> Vs;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int qtiles = max(1, (p.Lq + 63) / 64);
  const Work work = work_of_block(p, qtiles * p.cuts, p.H / p.G, true);
  if (work.none) return;
  const int b = work.b, h = work.h, kh = h / (p.H / p.G), cut = work.tile % p.cuts;
  if (b == p.B) {   // packed: rows of no sequence
    zero_rest<T>((T*)p.Oout, p.ldo, (int64_t)h * p.d, p.d, p.q_off, p.B, p.Tq, work.tile, TAIL);
    return;
  }
  const Seq sq = seq_of(p, b);
  const int i0 = work.tile / p.cuts * 64;
  if (i0 >= sq.Lq) return;   // block-uniform
  const int i = i0 + wave * 16 + c, pos = i + sq.off;
  KeySweep<T, D> keys(p, sq, b, kh, i0, cut, p.cuts);
  f32x4_t fq[D / 16], o[D / 16];
  load_own<T, D>(fq, (const T*)p.Q + (sq.qbase + min(i, sq.Lq - 1)) * p.ldq + (int64_t)h * p.d, p.d, g, i < sq.Lq);
#pragma unroll
  for (int t = 0; t < D / 16; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float cs = p.scale * LOG2E;   // scores in units of log 2: exp2 is one instruction, exp a dozen
  float m = -INFINITY, l = 0.f;
  for (int t = keys.beg; t < keys.end; ++t) {
    const uint64_t ok = keys.next(t, Ks, Vs), see = i < sq.Lq ? keys_seen(p, pos, keys.start(t), ok) : 0;
    const uint64_t mk = see >> (4 * g);
    f32x4_t sc[4];
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sc[k] = f32x4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (!piece(see, k)) continue;
      sc[k] = dot_rows<D>(Ks, 16 * k, fq, lane) * cs;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[k][r] = keep_or(sc[k][r], mk, k, r, 0xff800000u);   // -inf
        mx = fmaxf(mx, sc[k][r]);
      }
    }
    const float mn = fmaxf(m, quad_max(mx)), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - base);
    float rs = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sc[k][r] = __builtin_amdgcn_exp2f(sc[k][r] - base);
        rs += sc[k][r];
      }
    l = l * alpha + quad_sum(rs);
    m = mn;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) o[x] *= alpha;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (piece(see, k)) add_cols<D>(o, Vs, 16 * k, sc[k], lane);
  }
  if (p.cuts > 1) {
    if (i >= sq.Lq) return;
    const int64_t row = ((int64_t)cut * p.H + h) * p.Tq + sq.qbase + i;
    store_own<float, D>(p.cut_o + row * p.d, o, 1.f, p.d, g);
    if (g == 0) { p.cut_ml[2 * row] = m; p.cut_ml[2 * row + 1] = l; }
    return;
  }
  if (i < sq.Lq) {
    store_own<T, D>((T*)p.Oout + (sq.qbase + i) * p.ldo + (int64_t)h * p.d, o, l > 0.f || l != l ? 1.f / l : 0.f, p.d, g);
    if (g == 0) p.LSE[(int64_t)h * p.Tq + sq.qbase + i] = l > 0.f ? m * LN2 + logf(l) : (l != l ? l : -INFINITY);
  }
}

// ------------------------------------------------------------------------------ dQ, delta
template <typename T, int D>
__global__ __launch_bounds__(256, BLOCKS(D)) void window_dq_kernel(WinParams p) {
  __shared__ __attribute__((aligned(16))) Tile<D> Ks;
  __shared__ __attribute__((aligned(16))) Tile<D> Vs;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int qtiles = max(1, (p.Lq + 63) / 64);
  const Work work = work_of_block(p, qtiles * p.cuts, p.H / p.G, true);
  if (work.none) return;
  const int b = work.b, h = work.h, kh = h / (p.H / p.G), cut = work.tile % p.cuts;
  if (b == p.B) {
    zero_rest<T>((T*)p.dQ, p.lddq, (int64_t)h * p.d, p.d, p.q_off, p.B, p.Tq, work.tile, TAIL);
    return;
  }
  const Seq sq = seq_of(p, b);
  const int i0 = work.tile / p.cuts * 64;
  if (i0 >= sq.Lq) return;
  const int i = i0 + wave * 16 + c, pos = i + sq.off;
  const int64_t row = sq.qbase + min(i, sq.Lq - 1), si = (int64_t)h * p.Tq + row;
  KeySweep<T, D> keys(p, sq, b, kh, i0, cut, p.cuts);
  // bf16 rows of few keys: delta in fp32 from a sweep of its own, since O carries two roundings to 2^-8 (window_attn_mfma.hip)
  __shared__ int s_few[4][2];
  bool few_row = false, few = false;
  if constexpr (sizeof(T) == 2) {
    const FewKeys fk = few_keys(p, keys.kt, pos, i < sq.Lq, [&](int t) { return keys.padding(t); }, [&](int t, int no) { return keys.usable(t, no); });
    if (lane == 0) { s_few[wave][0] = fk.lo; s_few[wave][1] = fk.hi; }
    few_row = fk.row;
    few = __syncthreads_or(few_row);
  }
  f32x4_t fq[D / 16], fd[D / 16], dq[D / 16];
  load_own<T, D>(fq, (const T*)p.O + row * p.ldo + (int64_t)h * p.d, p.d, g, i < sq.Lq);
  load_own<T, D>(fd, (const T*)p.dO + row * p.lddo + (int64_t)h * p.d, p.d, g, i < sq.Lq);
  float dl = 0.f;
#pragma unroll
  for (int t = 0; t < D / 16; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) dl += fq[t][r] * fd[t][r];
    dq[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  dl = quad_sum(dl);
  load_own<T, D>(fq, (const T*)p.Q + row * p.ldq + (int64_t)h * p.d, p.d, g, i < sq.Lq);
  const float cs = p.scale * LOG2E, lse2 = p.LSE[si] * LOG2E;
  auto sweep = [&](auto delta_only) {
    float sum = 0.f;
    for (int t = keys.beg; t < keys.end; ++t) {
      const uint64_t ok = keys.next(t, Ks, Vs), see = i < sq.Lq ? keys_seen(p, pos, keys.start(t), ok) : 0;
      const uint64_t mk = see >> (4 * g);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (!piece(see, k)) continue;
        f32x4_t ds = dot_rows<D>(Ks, 16 * k, fq, lane);
        const f32x4_t dp = dot_rows<D>(Vs, 16 * k, fd, lane);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ds[r] = keep_or(__builtin_amdgcn_exp2f(fmaf(ds[r], cs, -lse2)) * (delta_only ? dp[r] : dp[r] - dl), mk, k, r, 0u);
          if (delta_only) sum += ds[r];
        }
        if constexpr (!delta_only) add_cols<D>(dq, Ks, 16 * k, ds, lane);
      }
    }
    return sum;
  };
  if constexpr (sizeof(T) == 2) {
    if (few) {
      const int beg = keys.beg, end = keys.end;
      keys.beg = min(min(s_few[0][0], s_few[1][0]), min(s_few[2][0], s_few[3][0]));
      keys.end = max(max(s_few[0][1], s_few[1][1]), max(s_few[2][1], s_few[3][1]));
      if (keys.beg < keys.end) keys.load(keys.beg);
      const float exact = quad_sum(sweep(std::true_type{}));
      dl = few_row ? exact : dl;
      keys.beg = beg;
      keys.end = end;
      if (beg < end) keys.load(beg);
    }
  }
  if (i < sq.Lq && g == 0 && cut == 0) p.delta[si] = dl;
  sweep(std::false_type{});
  if (p.cuts > 1) {
    if (i < sq.Lq) store_own<float, D>(p.cut_o + (((int64_t)cut * p.H + h) * p.Tq + row) * p.d, dq, p.scale, p.d, g);
    return;
  }
  if (i < sq.Lq) store_own<T, D>((T*)p.dQ + (sq.qbase + i) * p.lddq + (int64_t)h * p.d, dq, p.scale, p.d, g);
}

// ------------------------------------------------------------------------------ dK, dV
template <typename T, int D>
__global__ __launch_bounds__(256, BLOCKS(D)) void window_dkv_kernel(WinParams p) {
  __shared__ __attribute__((aligned(16))) Tile<D> Qs;
  __shared__ __attribute__((aligned(16))) Tile<D> Ds;
  __shared__ float s_lse[NT], s_dl[NT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int ktiles = max(1, (p.Lk + NT - 1) / NT);
  const Work work = work_of_block(p, key_tiles_of_grid(p, ktiles), 1, p.nst > 0);
  if (work.none) return;
  const int b = work.b, kh = work.h, rep = p.H / p.G;
  if (b == p.B) {
    zero_rest<T>((T*)p.dK, p.lddk, (int64_t)kh * p.d, p.d, p.k_off, p.B, p.Tk, work.tile, TAIL);
    zero_rest<T>((T*)p.dV, p.lddv, (int64_t)kh * p.d, p.d, p.k_off, p.B, p.Tk, work.tile, TAIL);
    return;
  }
  const Seq sq = seq_of(p, b);
  const KeyWork kw = key_work(p, ktiles, work.tile);
  const int tile = kw.tile, chunk = kw.chunk;
  const int j0 = tile * NT, j1 = min(j0 + NT, sq.Lk);
  if (j0 >= sq.Lk) return;
  int i_lo, i_hi;
  query_range(p, sq, j0, j1, chunk, i_lo, i_hi);
  if (chunk >= 0 && i_lo >= i_hi) return;   // (the join counts the same chunks)
  const int j = j0 + wave * 16 + c, jrow = min(j, sq.Lk - 1);
  const bool alive = j < sq.Lk && !(p.key_pad && p.key_pad[(int64_t)b * p.Lk + jrow]);
  const bool sink = p.nst && j < p.sinks;   // (a sink's sum has further parts)
  f32x4_t fk[D / 16], fv[D / 16], dk[D / 16], dv[D / 16];
  load_own<T, D>(fk, (const T*)p.K + (sq.kbase + jrow) * p.ldk + (int64_t)kh * p.d, p.d, g, alive);
  load_own<T, D>(fv, (const T*)p.V + (sq.kbase + jrow) * p.ldv + (int64_t)kh * p.d, p.d, g, alive);
#pragma unroll
  for (int t = 0; t < D / 16; ++t) dk[t] = dv[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int per = (i_hi - i_lo + NT - 1) / NT, n = per * rep;
  const float cs = p.scale * LOG2E;
  Stage<T, D> stage_q, stage_d;
  float row_lse = 0.f, row_dl = 0.f;
  auto load = [&](int t) {
    const int hh = t / per, r0 = i_lo + (t - hh * per) * NT, h = kh * rep + hh;
    stage_q.load((const T*)p.Q + sq.qbase * p.ldq + (int64_t)h * p.d, p.ldq, r0, sq.Lq, p.d, p.vec);
    stage_d.load((const T*)p.dO + sq.qbase * p.lddo + (int64_t)h * p.d, p.lddo, r0, sq.Lq, p.d, p.vec);
    const int64_t si = (int64_t)h * p.Tq + sq.qbase + min(r0 + (int)(threadIdx.x & 63), sq.Lq - 1);
    row_lse = p.LSE[si];
    row_dl = p.delta[si];
  };
  const int t_beg = chunk < 0 ? (int)((int64_t)n * kw.part / p.parts) : 0, t_end = chunk < 0 ? (int)((int64_t)n * (kw.part + 1) / p.parts) : n;
  if (t_beg < t_end) load(t_beg);
  for (int t = t_beg; t < t_end; ++t) {
    const int r0 = i_lo + (t % per) * NT;
    const uint64_t ok = bits(0, i_hi - r0);
    __syncthreads();
    stage_q.store(Qs, ok, p.d);
    stage_d.store(Ds, ok, p.d);
    if (threadIdx.x < NT) { s_lse[threadIdx.x] = row_lse * LOG2E; s_dl[threadIdx.x] = row_dl; }
    __syncthreads();
    if (t + 1 < t_end) load(t + 1);
    const uint64_t see = alive ? queries_seeing(p, j, r0 + sq.off, i_hi - r0) : 0;
    const uint64_t mk = see >> (4 * g);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!piece(see, k)) continue;
      f32x4_t pr = dot_rows<D>(Qs, 16 * k, fk, lane), ds = dot_rows<D>(Ds, 16 * k, fv, lane);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int il = 16 * k + 4 * g + r;
        const float e = __builtin_amdgcn_exp2f(fmaf(pr[r], cs, -s_lse[il]));
        ds[r] = keep_or(e * (ds[r] - s_dl[il]), mk, k, r, 0u);
        pr[r] = keep_or(e, mk, k, r, 0u);
      }
      add_cols<D>(dv, Ds, 16 * k, pr, lane);
      add_cols<D>(dk, Qs, 16 * k, ds, lane);
    }
  }
  if (j >= sq.Lk) return;
  if (p.parts > 1 && chunk < 0) {
    store_own<float, D>(split_row(p, kw.part, 0, b, j, kh), dk, p.scale, p.d, g);
    store_own<float, D>(split_row(p, kw.part, 1, b, j, kh), dv, 1.f, p.d, g);
  } else if (sink) {
    float* s = slab(p, b, kh, tile, 1 + chunk, NT) + (int64_t)(j - j0) * p.d;
    store_own<float, D>(s, dk, p.scale, p.d, g);
    store_own<float, D>(s + (int64_t)slab_rows(p, NT) * p.d, dv, 1.f, p.d, g);
  } else if (chunk < 0) {
    store_own<T, D>((T*)p.dK + (sq.kbase + j) * p.lddk + (int64_t)kh * p.d, dk, p.scale, p.d, g);
    store_own<T, D>((T*)p.dV + (sq.kbase + j) * p.lddv + (int64_t)kh * p.d, dv, 1.f, p.d, g);
  }
}

// dK, dV of the sinks: window part and chunks added in this order.  `rows`: key rows of a tile.
template <typename T>
__global__ __launch_bounds__(256) void window_join_kernel(WinParams p, int rows) {
  const int b = blockIdx.z, kh = blockIdx.y;
  const Seq sq = seq_of(p, b);
  const int e = (int)blockIdx.x * 256 + threadIdx.x, j = e / p.d, c = e - j * p.d;
  if (j >= min(p.sinks, sq.Lk)) return;
  const int tile = j / rows, j0 = tile * rows;
  int lo, hi, parts = 1;
  query_range(p, sq, j0, min(j0 + rows, sq.Lk), 0, lo, hi);
  if (lo < hi) parts += (sq.Lq - lo + p.ch - 1) / p.ch;
  const float* x = slab(p, b, kh, tile, 0, rows) + (int64_t)(j - j0) * p.d + c;
  const int64_t half = (int64_t)slab_rows(p, rows) * p.d, step = 2 * half;
  float a = 0.f, v = 0.f;
#pragma unroll 8
  for (int s = 0; s < parts; ++s) {
    a += x[s * step];
    v += x[s * step + half];
  }
  ((T*)p.dK)[(sq.kbase + j) * p.lddk + (int64_t)kh * p.d + c] = Cvt<T>::from_f32(a);
  ((T*)p.dV)[(sq.kbase + j) * p.lddv + (int64_t)kh * p.d + c] = Cvt<T>::from_f32(v);
}

// dK, dV of all keys where windows are cut into parts: the parts, then a sink's chunks.
template <typename T>
__global__ __launch_bounds__(256) void window_split_join_kernel(WinParams p, int rows) {
  const int b = blockIdx.y;
  const Seq sq = seq_of(p, b);
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int width = p.G * p.d, j = (int)(e / width), col = (int)(e - (int64_t)j * width), kh = col / p.d, c = col - kh * p.d;
  if (j >= sq.Lk) return;
  const float* x = split_row(p, 0, 0, b, j, kh) + c;
  const int64_t half = (int64_t)p.B * p.Lk * width;
  float a = 0.f, v = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.parts; ++s) {
    a += x[2 * s * half];
    v += x[(2 * s + 1) * half];
  }
  if (p.nst && j < p.sinks) {
    const int tile = j / rows, j0 = tile * rows;
    int lo, hi;
    query_range(p, sq, j0, min(j0 + rows, sq.Lk), 0, lo, hi);
    const int chunks = lo < hi ? (sq.Lq - lo + p.ch - 1) / p.ch : 0;
    for (int s = 1; s <= chunks; ++s) {
      const float* y = slab(p, b, kh, tile, s, rows) + (int64_t)(j - j0) * p.d + c;
      a += y[0];
      v += y[(int64_t)slab_rows(p, rows) * p.d];
    }
  }
  ((T*)p.dK)[(sq.kbase + j) * p.lddk + col] = Cvt<T>::from_f32(a);
  ((T*)p.dV)[(sq.kbase + j) * p.lddv + col] = Cvt<T>::from_f32(v);
}

// O and log-sum-exp of rows whose keys were cut: a thread per element.
template <typename T>
__global__ __launch_bounds__(256) void window_cut_join_kernel(WinParams p) {
  const int b = blockIdx.y, width = p.H * p.d;
  const Seq sq = seq_of(p, b);
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(e / width), col = (int)(e - (int64_t)i * width), h = col / p.d, c = col - h * p.d;
  if (i >= sq.Lq) return;
  const int64_t row = (int64_t)h * p.Tq + sq.qbase + i, step = (int64_t)p.H * p.Tq;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int s = 0; s < p.cuts; ++s) m = fmaxf(m, p.cut_ml[2 * (row + s * step)]);
#pragma unroll 4
  for (int s = 0; s < p.cuts; ++s) {
    const float2 ml = *(const float2*)&p.cut_ml[2 * (row + s * step)];
    const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(ml.x - m);   // (a sum of NaN scores has no maximum)
    l += f * ml.y;
    o += f * p.cut_o[(row + s * step) * p.d + c];
  }
  const bool some = l > 0.f || l != l;
  ((T*)p.Oout)[(sq.qbase + i) * p.ldo + col] = Cvt<T>::from_f32(some ? o / l : 0.f);
  if (c == 0) p.LSE[row] = l > 0.f ? m * LN2 + logf(l) : (some ? l : -INFINITY);
}

// dQ of rows whose keys were cut.
template <typename T>
__global__ __launch_bounds__(256) void window_cut_sum_kernel(WinParams p) {
  const int b = blockIdx.y, width = p.H * p.d;
  const Seq sq = seq_of(p, b);
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int i = (int)(e / width), col = (int)(e - (int64_t)i * width), h = col / p.d, c = col - h * p.d;
  if (i >= sq.Lq) return;
  const float* x = p.cut_o + ((int64_t)h * p.Tq + sq.qbase + i) * p.d + c;
  float a = 0.f;
#pragma unroll 8
  for (int s = 0; s < p.cuts; ++s) a += x[(int64_t)s * p.H * p.Tq * p.d];
  ((T*)p.dQ)[(sq.qbase + i) * p.lddq + col] = Cvt<T>::from_f32(a);
}

// whether every row of the operands that go through LDS is made of whole 4-element pieces
bool whole_pieces(const WinParams& p, int dtype) {
  const int64_t size = dtype == SK_BF16 ? 2 : 4;
  return p.d % 4 == 0 && (p.ldq | p.ldk | p.ldv | p.lddo) % 4 == 0 &&
         (((uintptr_t)p.Q | (uintptr_t)p.K | (uintptr_t)p.V | (uintptr_t)p.dO) & (4 * size - 1)) == 0;
}

int check(const char* who, const WinParams& p, int window, int dtype) {
  SK_CHECK_ARG(dtype == SK_F32 || dtype == SK_BF16, "%s: bad dtype %d", who, dtype);
  SK_CHECK_ARG(p.B >= 0 && p.H > 0 && p.G > 0 && p.Lq >= 0 && p.Lk >= 0 && p.Tq >= 0 && p.Tk >= 0, "%s: bad shape", who);
  SK_CHECK_ARG(p.H % p.G == 0, "%s: %d query heads do not share %d key heads evenly", who, p.H, p.G);
  SK_CHECK_ARG(p.d > 0 && p.d <= MAXD, "%s: head size %d must be in 1..%d", who, p.d, MAXD);
  SK_CHECK_ARG(p.H <= 65535 && p.B <= 65534, "%s: more than 65535 heads or 65534 sequences", who);
  SK_CHECK_ARG(p.Lq <= MAX_LEN && p.Lk <= MAX_LEN, "%s: sequences of more than 2^29 positions", who);
  SK_CHECK_ARG(window >= 1 && p.sinks >= 0, "%s: window %d must be >= 1 and sinks %d >= 0", who, window, p.sinks);
  SK_CHECK_ARG(!p.q_off == !p.k_off, "%s: one offset array without the other", who);
  SK_CHECK_ARG(!(p.q_off && p.key_pad), "%s: packed rows take no padding mask", who);
  SK_CHECK_ARG(p.q_off || (p.Tq == (int64_t)p.B * p.Lq && p.Tk == (int64_t)p.B * p.Lk), "%s: rows are not B x L", who);
  const int64_t nq = (int64_t)p.H * p.d, nk = (int64_t)p.G * p.d;
  SK_CHECK_ARG(p.ldq >= nq && p.ldo >= nq && p.ldk >= nk && p.ldv >= nk, "%s: row stride below the row's length", who);
  return SK_OK;
}

void set_window(WinParams& p, int window, int causal) {
  const int span = p.Lq + p.Lk;
  p.left = std::min(window - 1, span);
  p.right = causal ? 0 : p.left;
  if (p.sinks >= p.Lk) p.left = span;   // every key stays visible
  p.sinks = std::min(p.sinks, p.Lk);
}

int64_t slab_floats(const WinParams& p, int rows) {
  return ((int64_t)p.B * p.G * p.nst * (1 + p.nch) * 2 * slab_rows(p, rows) * p.d + 3) / 4 * 4;   // (16-byte stores behind)
}

// Parts of a key tile's window: two blocks for every CU, each with at least four tiles of queries (bf16, 2 x 4096 tokens, 8
// heads of 128 over 2 key heads, window 512: 128 blocks alone 178 us, cut in four 80 and 15 for the join; fp32, 3 x 2000
// tokens, 4 heads of 96 over one, window 1024, 30 sinks: 945 and 440).
// Tiles that hold sinks and the chunks their far queries are cut into: about as many rows per chunk as a part of a key
// tile's own window has, so that these blocks last no longer than the others.
void plan_keys(WinParams& p, int rows) {
  const int64_t cus = sk_num_cus(), units = (int64_t)p.B * p.G, blocks = std::max<int64_t>(1, units * ((p.Lk + rows - 1) / rows));
  const int64_t span = (int64_t)p.left + p.right + rows, tiles = (std::min<int64_t>(p.Lq, span) + 63) / 64 * (p.H / p.G);
  p.parts = (int)std::max<int64_t>(1, std::min(2 * cus / blocks, tiles / 4));
  const bool far = p.sinks > 0 && p.left < p.Lk;   // else every query's window reaches key 0
  p.nst = far ? (p.sinks + rows - 1) / rows : 0;
  p.ch = (int)std::max<int64_t>(256, (span + 63) / 64 * 64);
  const int64_t less = std::max<int64_t>(64, (span / p.parts + 63) / 64 * 64);
  if (units * p.nst * (p.Lq / less + 1) <= 4 * cus) p.ch = (int)std::min<int64_t>(p.ch, p.parts > 1 ? less : p.ch);
  p.nch = far ? (p.Lq + p.ch - 1) / p.ch : 0;
  // The sums in memory grow with sinks x Lq / ch.  Where they are large the sink tiles are many, and four blocks for every CU
  // do: longer chunks, and no chunks where the tiles alone are that many (their blocks sweep the far queries too, query_range).
  // At most 4096 x rows x d floats then remain, however many sinks (32768 tokens, 8 heads of 128, window 64, 4096 sinks:
  // 4.3 GB -> 168 MB).
  if (slab_floats(p, rows) <= 1 << 24) return;
  const int64_t most = 4 * cus / (units * p.nst);
  if (most >= 1) {
    p.ch = std::max<int64_t>(p.ch, ((p.Lq + most - 1) / most + 63) / 64 * 64);
    p.nch = (p.Lq + p.ch - 1) / p.ch;
  } else {
    p.nst = p.nch = 0;
  }
}

// Cuts of a query tile's keys: two blocks for every CU, each with at least 12 tiles of 64 keys (fp32 arithmetic: 8).  64
// queries at the end of 32768 keys, 8 heads of 128, all visible: 8 blocks alone 649 us, cut 46, with the backward pass 1262
// and 172 (fp32 4276 and 144, 5861 and 724); 4096 tokens, 4 heads of 64, causal: 74 and 36.  Shorter sweeps are not worth
// the join: 2048 tokens, 8 heads of 128, window 1024 (18 tiles): uncut 30, in two 38.
// (Partial outputs are kept for every row of Q: a packed tensor with more rows than its sequences counts whole.)
void plan_cuts(WinParams& p, int rows) {
  const int64_t blocks = std::max<int64_t>({1, (int64_t)p.B * p.H * ((p.Lq + rows - 1) / rows), p.H * p.Tq / rows});
  const int64_t tiles = std::min<int64_t>(p.Lk, (int64_t)rows + p.left + p.right + p.sinks) / 64;
  p.cuts = (int)std::max<int64_t>(1, std::min({2 * (int64_t)sk_num_cus() / blocks, tiles / (rows == NT ? 8 : 12), (int64_t)64}));
}
int64_t cut_o_floats(const WinParams& p) { return ((int64_t)p.cuts * p.H * p.Tq * p.d + 3) / 4 * 4; }
int64_t cut_floats(const WinParams& p) { return p.cuts > 1 ? cut_o_floats(p) + 2ll * p.cuts * p.H * p.Tq : 0; }

// Grids of 256 threads a block whose threads are counted in 32 bits (tiles of 64 rows: the most that any kernel has).
bool grids_fit(const WinParams& p) {
  const int64_t tiles = std::max(p.Lq, p.Lk) / 64 + 1, units = (int64_t)p.B * p.G + 7;
  return units * tiles * std::max(1, p.cuts) * (p.H / p.G) + TAIL * p.H < (1 << 24) && units * (tiles * p.parts + (int64_t)p.nst * p.nch) + TAIL * p.G < (1 << 24) &&
         (p.nst == 0 || (int64_t)p.sinks * p.d < (1ll << 31));
}

int64_t split_floats(const WinParams& p) { return p.parts > 1 ? 2ll * p.parts * p.B * p.Lk * p.G * p.d : 0; }

template <typename T, int D>
void launch_fwd_at(const WinParams& p, hipStream_t stream) {
  const dim3 grid(work_blocks(p, std::max(1, (p.Lq + 63) / 64) * p.cuts, p.H / p.G));
  hipLaunchKernelGGL((window_fwd_kernel<T, D>), grid, dim3(256), 0, stream, p);
}
template <typename T, int D>
void launch_bwd_at(const WinParams& p, hipStream_t stream) {
  const dim3 gq(work_blocks(p, std::max(1, (p.Lq + 63) / 64) * p.cuts, p.H / p.G));
  const dim3 gk(work_blocks(p, key_tiles_of_grid(p, std::max(1, (p.Lk + NT - 1) / NT)), 1));
  if (p.Tq) hipLaunchKernelGGL((window_dq_kernel<T, D>), gq, dim3(256), 0, stream, p);
  if (p.Tk) hipLaunchKernelGGL((window_dkv_kernel<T, D>), gk, dim3(256), 0, stream, p);
}
// Heads are computed at the next multiple of 32 elements (4 x 4096 tokens, 8 heads, window 512, forward and backward: 32 of
// 64 columns 862 us, of 32 466; 80 of 128 2540, of 96 1570).
template <typename T>
void launch_fwd(const WinParams& p, hipStream_t stream) {
  if (p.d <= 32) launch_fwd_at<T, 32>(p, stream);
  else if (p.d <= 64) launch_fwd_at<T, 64>(p, stream);
  else if (p.d <= 96) launch_fwd_at<T, 96>(p, stream);
  else launch_fwd_at<T, 128>(p, stream);
}
template <typename T>
void launch_bwd(const WinParams& p, hipStream_t stream) {
  if (p.d <= 32) launch_bwd_at<T, 32>(p, stream);
  else if (p.d <= 64) launch_bwd_at<T, 64>(p, stream);
  else if (p.d <= 96) launch_bwd_at<T, 96>(p, stream);
  else launch_bwd_at<T, 128>(p, stream);
}

}  // namespace

int sk_window_join(const WinParams& p, int rows, int dtype, hipStream_t stream) {
  if (p.cuts > 1 && p.B && p.Lq) {
    const dim3 all((unsigned)(((int64_t)p.Lq * p.H * p.d + 255) / 256), p.B);
    if (dtype == SK_BF16) hipLaunchKernelGGL((window_cut_sum_kernel<bf16_t>), all, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((window_cut_sum_kernel<float>), all, dim3(256), 0, stream, p);
    SK_CHECK_LAUNCH("skhip_window_attn_bwd(join)");
  }
  if ((!p.nst && p.parts == 1) || !p.B || !p.Lk) return SK_OK;   // (no sequence has keys: no grid)
  if (p.parts > 1) {
    const dim3 all((unsigned)(((int64_t)p.Lk * p.G * p.d + 255) / 256), p.B);
    if (dtype == SK_BF16) hipLaunchKernelGGL((window_split_join_kernel<bf16_t>), all, dim3(256), 0, stream, p, rows);
    else hipLaunchKernelGGL((window_split_join_kernel<float>), all, dim3(256), 0, stream, p, rows);
    SK_CHECK_LAUNCH("skhip_window_attn_bwd(join)");
    return SK_OK;
  }
  dim3 grid((unsigned)(((int64_t)p.sinks * p.d + 255) / 256), p.G, p.B);
  if (dtype == SK_BF16) hipLaunchKernelGGL((window_join_kernel<bf16_t>), grid, dim3(256), 0, stream, p, rows);
  else hipLaunchKernelGGL((window_join_kernel<float>), grid, dim3(256), 0, stream, p, rows);
  SK_CHECK_LAUNCH("skhip_window_attn_bwd(join)");
  return SK_OK;
}

int sk_window_cut_join(const WinParams& p, int dtype, hipStream_t stream) {
  if (p.cuts == 1 || !p.B || !p.Lq) return SK_OK;   // (no sequence has queries: no grid)
  const dim3 all((unsigned)(((int64_t)p.Lq * p.H * p.d + 255) / 256), p.B);
  if (dtype == SK_BF16) hipLaunchKernelGGL((window_cut_join_kernel<bf16_t>), all, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((window_cut_join_kernel<float>), all, dim3(256), 0, stream, p);
  SK_CHECK_LAUNCH("skhip_window_attn_fwd(join)");
  return SK_OK;
}

// sizes that a call would take (the size queries answer 0 for others)
static bool sizes_fit(int B, int n_head, int n_kv, int64_t Tq, int Lq, int Lk, int d, int window, int sinks) {
  return B >= 0 && n_head > 0 && n_kv > 0 && n_head % n_kv == 0 && Tq >= 0 && Lq >= 0 && Lq <= MAX_LEN && Lk >= 0 && Lk <= MAX_LEN &&
         d > 0 && d <= MAXD && window >= 1 && sinks >= 0;
}

extern "C" int64_t skhip_window_attn_fwd_ws_floats(int B, int n_head, int n_kv, int64_t Tq, int Lq, int Lk, int d, int window,
                                                   int sinks, int causal) {
  if (!sizes_fit(B, n_head, n_kv, Tq, Lq, Lk, d, window, sinks)) return 0;
  WinParams p = {};
  p.B = B; p.H = n_head; p.G = n_kv; p.Tq = Tq; p.Lq = Lq; p.Lk = Lk; p.d = d; p.sinks = sinks;
  set_window(p, window, causal);
  // the larger of the two paths' needs: which one a call takes depends on its pointers and strides
  plan_cuts(p, NT);
  const int64_t plain = cut_floats(p);
  plan_cuts(p, MFMA_ROWS);
  return std::max(plain, cut_floats(p));
}

extern "C" int64_t skhip_window_attn_bwd_ws_floats(int B, int n_head, int n_kv, int64_t Tq, int Lq, int Lk, int d, int window,
                                                   int sinks, int causal) {
  if (!sizes_fit(B, n_head, n_kv, Tq, Lq, Lk, d, window, sinks)) return 0;
  WinParams p = {};
  p.B = B; p.H = n_head; p.G = n_kv; p.Tq = Tq; p.Lq = Lq; p.Lk = Lk; p.d = d; p.sinks = sinks;
  set_window(p, window, causal);
  // the larger of the two paths' needs: which one a call takes depends on its pointers and strides
  plan_keys(p, NT);
  plan_cuts(p, NT);
  const int64_t plain = ((int64_t)n_head * Tq + 3) / 4 * 4 + slab_floats(p, NT) + split_floats(p) + cut_floats(p);
  plan_keys(p, MFMA_ROWS);
  plan_cuts(p, MFMA_ROWS);
  return std::max(plain, (2 * (int64_t)n_head * Tq + 3) / 4 * 4 + slab_floats(p, MFMA_ROWS) + split_floats(p) + cut_floats(p));
}

extern "C" int skhip_window_attn_fwd(const void* Q, const void* K, const void* V, void* O, float* LSE, const uint8_t* key_pad,
                                     const int32_t* q_off, const int32_t* k_off, int B, int n_head, int n_kv, int64_t Tq,
                                     int64_t Tk, int Lq, int Lk, int d, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo,
                                     float scale, int window, int sinks, int causal, float* workspace,
                                     int64_t workspace_floats, int dtype, void* stream_) {
  const char* who = "skhip_window_attn_fwd";
  hipStream_t stream = (hipStream_t)stream_;
  WinParams p = {};
  p.Q = Q; p.K = K; p.V = V; p.Oout = O; p.LSE = LSE; p.key_pad = key_pad; p.q_off = q_off; p.k_off = k_off;
  p.B = B; p.H = n_head; p.G = n_kv; p.Tq = Tq; p.Tk = Tk; p.Lq = Lq; p.Lk = Lk; p.d = d;
  p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo; p.scale = scale; p.sinks = sinks;
  int rc = check(who, p, window, dtype);
  if (rc) return rc;
  if (Tq == 0) return SK_OK;
  SK_CHECK_ARG(Q && O && LSE && (Tk == 0 || (K && V)), "%s: null pointer", who);
  set_window(p, window, causal);
  const bool mfma = sk_window_mfma_supported(p, dtype);
  plan_cuts(p, mfma ? MFMA_ROWS : NT);
  SK_CHECK_ARG(grids_fit(p), "%s: more than 2^24 tiles of 64 rows", who);
  const int64_t need = cut_floats(p);
  if (need > 0 && (!workspace || workspace_floats < need)) {
    sk_set_error("%s: workspace of %lld floats needed", who, (long long)need);
    return SK_ERR_WORKSPACE;
  }
  SK_CHECK_ARG(need == 0 || ((uintptr_t)workspace & 15) == 0, "%s: workspace not aligned to 16 bytes", who);
  p.cut_o = workspace;
  p.cut_ml = workspace + cut_o_floats(p);
  if (mfma) {
    rc = sk_window_fwd_mfma(p, stream);
    return rc ? rc : sk_window_cut_join(p, dtype, stream);
  }
  p.vec = whole_pieces(p, dtype);
  if (dtype == SK_BF16) {
    launch_fwd<bf16_t>(p, stream);
  } else {
    launch_fwd<float>(p, stream);
  }
  SK_CHECK_LAUNCH(who);
  return sk_window_cut_join(p, dtype, stream);
}

extern "C" int skhip_window_attn_bwd(const void* Q, const void* K, const void* V, const void* O, const void* dO,
                                     const float* LSE, void* dQ, void* dK, void* dV, const uint8_t* key_pad,
                                     const int32_t* q_off, const int32_t* k_off, int B, int n_head, int n_kv, int64_t Tq,
                                     int64_t Tk, int Lq, int Lk, int d, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo,
                                     int64_t lddo, int64_t lddq, int64_t lddk, int64_t lddv, float scale, int window,
                                     int sinks, int causal, float* workspace, int64_t workspace_floats, int dtype,
                                     void* stream_) {
  const char* who = "skhip_window_attn_bwd";
  hipStream_t stream = (hipStream_t)stream_;
  WinParams p = {};
  p.Q = Q; p.K = K; p.V = V; p.O = O; p.dO = dO; p.LSE = (float*)LSE; p.dQ = dQ; p.dK = dK; p.dV = dV;
  p.key_pad = key_pad; p.q_off = q_off; p.k_off = k_off;
  p.B = B; p.H = n_head; p.G = n_kv; p.Tq = Tq; p.Tk = Tk; p.Lq = Lq; p.Lk = Lk; p.d = d;
  p.ldq = ldq; p.ldk = ldk; p.ldv = ldv; p.ldo = ldo; p.lddo = lddo; p.lddq = lddq; p.lddk = lddk; p.lddv = lddv;
  p.scale = scale; p.sinks = sinks;
  int rc = check(who, p, window, dtype);
  if (rc) return rc;
  const int64_t nq = (int64_t)n_head * d, nk = (int64_t)n_kv * d;
  SK_CHECK_ARG(lddo >= nq && lddq >= nq && lddk >= nk && lddv >= nk, "%s: row stride below the row's length", who);
  if (Tq == 0 && Tk == 0) return SK_OK;
  SK_CHECK_ARG((Tq == 0 || (Q && O && dO && LSE && dQ)) && (Tk == 0 || (K && V && dK && dV)), "%s: null pointer", who);
  set_window(p, window, causal);
  const bool mfma = sk_window_mfma_supported(p, dtype);
  const int rows = mfma ? MFMA_ROWS : NT;
  plan_keys(p, rows);
  plan_cuts(p, rows);
  SK_CHECK_ARG(grids_fit(p), "%s: more than 2^24 tiles of 64 rows", who);
  const int64_t head = (mfma ? 2 : 1) * (int64_t)n_head * Tq, need = (head + 3) / 4 * 4 + slab_floats(p, rows) + split_floats(p) + cut_floats(p);
  if (need > 0 && (!workspace || workspace_floats < need)) {
    sk_set_error("%s: workspace of %lld floats needed", who, (long long)need);
    return SK_ERR_WORKSPACE;
  }
  SK_CHECK_ARG(need == 0 || ((uintptr_t)workspace & 15) == 0, "%s: workspace not aligned to 16 bytes", who);
  p.delta = workspace;
  p.slabs = workspace + (head + 3) / 4 * 4;   // (16-byte stores)
  p.split = p.slabs + slab_floats(p, rows);
  p.cut_o = p.split + split_floats(p);   // (multiples of 4 floats up to here where 16-byte stores are made: d % 8 == 0)
  p.vec = whole_pieces(p, dtype);
  if (mfma) {
    rc = sk_window_bwd_mfma(p, stream);
    return rc ? rc : sk_window_join(p, rows, dtype, stream);
  }
  if (dtype == SK_BF16) {
    launch_bwd<bf16_t>(p, stream);
  } else {
    launch_bwd<float>(p, stream);
  }
  SK_CHECK_LAUNCH(who);
  return sk_window_join(p, rows, dtype, stream);
}
