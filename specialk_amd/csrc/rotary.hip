// Rotary positions of query and key heads, with an optional RMS norm of every head in the same pass, forward and backward.
//
// A head vector x of d elements at position p leaves as  y = R(p) N(x):
//   N(x) = x * rstd * gamma, rstd = 1 / sqrt(mean(x^2) + eps)      (identity without the norm)
//   R(p) turns rot / 2 pairs (a, b) of the first rot elements by the angles p f_i and scales them by A:
//        a' = A (a cos - b sin),  b' = A (b cos + a sin);           elements rot .. d-1 pass through.
// Pairs are (i, i + rot/2) or, interleaved, (2i, 2i + 1).  Backward, with g = R(p)^T dy (the same turn by -p f_i):
//   dgamma = sum over rows and heads of g * xhat, xhat = x * rstd;   dx = rstd (g gamma - xhat mean(g gamma xhat)).
// Without the norm backward IS the forward kernel with the angles negated.
//
// Angles: a frequency is a 64-bit fraction of a turn, so  position * frequency mod 2^64  is the exact phase at that frequency
// of any 64-bit position in one integer product (in 32-bit floats position 10^6 would already be off by 0.06 rad).  Its top bits give
// the quadrant and a remainder of at most 1/8 turn, which the Taylor polynomials of sine and cosine take to fp32
// accuracy.  A block computes the (cos, sin) of its tokens once into LDS and uses them for all heads.
//
// Bound by HBM: each element is read and written once (backward of the norm reads x and dy).  A lane owns 8 pairs, or 16
// of the elements that pass, of one head: two 16-byte loads and stores in bf16, no exchange between lanes but the
// norm's sum over the lanes of a head.  Many waves with one item each in flight carry more than few with several: against
// four items a thread (two backward) at 150 - 176 registers, one item at 60 - 128 takes norm and turn of 65536 rows of 40
// heads of 128 in bf16 from 280 to 250 us (5.4 TB/s), their backward from 451 to 430 us (4.7 TB/s, three passes over the
// rows), and the turn alone of 16381 rows of 20 fp32 heads of 128 from 90 to 75 us (4.5 TB/s); a copy reaches 4.9 TB/s.
#include "common.h"
#include <algorithm>

namespace {

constexpr int MAX_D = 256;        // at most 16 + 1 owning lanes per head
constexpr int ANGLES = 2048;      // (cos, sin) pairs per group of tokens
constexpr int BWD_BLOCKS = 1024;  // partial dgamma rows of the backward pass, queries and keys together

// Queries and keys are two sides of a launch, each with blocks of its own: a block then has one set of pointers, one norm
// weight and one gradient sum.
struct Side {
  const void *x, *dy;       // input (backward: the saved one), output gradient
  void* out;                // forward: output; backward: input gradient
  int64_t ldx, lddy, ldo;
  const float* gamma;       // [d]
  float* partial;           // [blocks][d]
  int64_t groups;           // of tb tokens
  int heads, tb, width, blocks;   // width: items (lanes of heads) per token
  uint32_t magic;                 // ceil(2^32 / width)
};
struct RotParams {
  Side side[2];
  const int64_t* pos;
  const uint64_t* turns;    // [rot / 2]
  int64_t T;
  int d, rot, lph;          // lanes per head (power of two)
  float amp, eps;
  int sign;                 // -1: angles negated
};

// cos and sin of 2 pi * phase / 2^64
__device__ __forceinline__ float2 turn_cos_sin(uint64_t phase) {
  const uint64_t ph = phase + (1ull << 61);
  const int quad = (int)(ph >> 62);
  const int32_t v = (int32_t)((uint32_t)(ph >> 30) ^ 0x80000000u);   // remainder in 2^-31 of an eighth of a turn
  const float x = (float)v * (0.78539816339744831f / 2147483648.f);
  const float z = x * x;
  // Taylor series about 0 for |x| <= pi / 4: the first terms left out are below 2e-9 (sine) and 2e-9 (cosine)
  const float s = x + x * z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880))));
  const float c = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 + z * (-1.f / 3628800)))));
  float2 r;
  r.x = (quad & 1) ? s : c;
  r.y = (quad & 1) ? c : s;
  if (quad == 1 || quad == 2) r.x = -r.x;
  if (quad >= 2) r.y = -r.y;
  return r;
}

// How the elements of a head are dealt to its lanes.
//  PAIRS     lane l holds 8 pairs, v[j] and v[8 + j] = the two halves of pair 8 l + j, or 16 consecutive passing elements;
//            16-byte loads where rot and d are multiples of 16.
//  ELEMENTS  lane l holds elements 16 l .. 16 l + 15, loaded 16 bytes at a time whatever rot is (d a multiple of 8); the other
//            half of a pair may lie with another lane of the head and is fetched through LDS.
//  SCALARS   the pairs, element by element: odd sizes and rows that are not 16-byte aligned.
// (46626 rows of 4 + 1 bf16 heads of 64, 36 elements turned, forward and backward: SCALARS 131 us, ELEMENTS 47.)
enum Deal { SCALARS, PAIRS, ELEMENTS };

template <typename T, bool IL, Deal DEAL>
struct Own {
  static constexpr int VN = Vec16<T>::N;
  static constexpr bool VEC = DEAL == PAIRS, ELEM = DEAL == ELEMENTS;
  static __device__ __forceinline__ int lanes(const RotParams& p) {
    return ELEM ? (p.d + 15) >> 4 : (((p.rot >> 1) + 7) >> 3) + ((p.d - p.rot + 15) >> 4);
  }
  static __device__ __forceinline__ int index(const RotParams& p, int l, int j) {   // j in 0 .. 15; -1: no element
    if (ELEM) return 16 * l + j < p.d ? 16 * l + j : -1;
    const int np = p.rot >> 1, nrl = (np + 7) >> 3;
    if (l < nrl) {
      const int pr = 8 * l + (j & 7);
      if (pr >= np) return -1;
      return IL ? 2 * pr + (j >> 3) : pr + (j >> 3) * np;
    }
    const int e = p.rot + 16 * (l - nrl) + j;
    return e < p.d ? e : -1;
  }
  // base: the head's first element.  Vector form (rot and d multiples of 16, 16-byte rows): two runs of 8 elements.
  static __device__ __forceinline__ int run(const RotParams& p, int l, int half) {
    if (ELEM) return 16 * l + 8 * half;
    const int np = p.rot >> 1, nrl = np >> 3;
    if (l < nrl) return IL ? 16 * l + 8 * half : 8 * l + half * np;
    return p.rot + 16 * (l - nrl) + 8 * half;
  }
  // raw[] is the lane's data as loaded
  typedef decltype(Vec16<T>().v) raw_t;
  static constexpr int NR = 16 / VN;
  struct Raw { raw_t r[NR]; };
  static __device__ __forceinline__ void load(Raw& w, const T* base, const RotParams& p, int l, bool active) {
    if constexpr (VEC || ELEM) {
      if (active) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < NR / 2; ++i)
            w.r[h * (NR / 2) + i] = !ELEM || run(p, l, h) < p.d ? *(const raw_t*)(base + run(p, l, h) + i * VN) : raw_t{};
      }
    } else {
      T* e = (T*)w.r;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = active ? index(p, l, j) : -1;
        e[j] = i >= 0 ? base[i] : Cvt<T>::from_f32(0.f);
      }
    }
  }
  // raw order -> pair order (v[j], v[8 + j] = pair j)
  static __device__ __forceinline__ void unpack(float (&v)[16], const Raw& w, bool rotates) {
    const T* e = (const T*)w.r;
    if (VEC && IL && rotates) {
#pragma unroll
      for (int j = 0; j < 8; ++j) { v[j] = Cvt<T>::to_f32(e[2 * j]); v[8 + j] = Cvt<T>::to_f32(e[2 * j + 1]); }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = Cvt<T>::to_f32(e[j]);
    }
  }
  static __device__ __forceinline__ void store(T* base, const float (&v)[16], const RotParams& p, int l, bool rotates) {
    if constexpr (VEC || ELEM) {
      Raw w;
      T* e = (T*)w.r;
      if (VEC && IL && rotates) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { e[2 * j] = Cvt<T>::from_f32(v[j]); e[2 * j + 1] = Cvt<T>::from_f32(v[8 + j]); }
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) e[j] = Cvt<T>::from_f32(v[j]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < NR / 2; ++i)
          if (!ELEM || run(p, l, h) < p.d) *(raw_t*)(base + run(p, l, h) + i * VN) = w.r[h * (NR / 2) + i];
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = index(p, l, j);
        if (i >= 0) base[i] = Cvt<T>::from_f32(v[j]);
      }
    }
  }
  // fp32 row vector of d elements (gamma) in pair order
  static __device__ __forceinline__ void load_row(float (&v)[16], const float* g, const RotParams& p, int l, bool rotates) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      int i;
      if constexpr (VEC) {
        if (IL && rotates) i = 16 * l + 2 * (j & 7) + (j >> 3);
        else i = run(p, l, j >> 3) + (j & 7);
        if (i >= p.d) i = -1;
      } else {
        i = index(p, l, j);
      }
      v[j] = i >= 0 ? g[i] : 0.f;
    }
  }
};

__device__ __forceinline__ void group_angles(float2* cs, const RotParams& p, int64_t t0, int nt) {
  const int np = p.rot >> 1;
  for (int e = threadIdx.x; e < nt * np; e += 256) {
    const int t = e / np, i = e - t * np;
    const int64_t ps = p.pos[t0 + t];
    float2 r = turn_cos_sin((uint64_t)ps * p.turns[i]);
    r.x *= p.amp;
    r.y *= p.sign < 0 ? -p.amp : p.amp;
    cs[e] = r;
  }
}

__device__ __forceinline__ float head_sum(float v, int lph) {
  for (int o = lph >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// dir > 0: a' = a cos - b sin ...; dir < 0: the turn back
template <int DIR>
__device__ __forceinline__ void turn(float (&v)[16], const float2* cs, int valid) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j >= valid) break;
    const float2 t = cs[j];
    const float a = v[j], b = v[8 + j];
    v[j] = DIR > 0 ? a * t.x - b * t.y : a * t.x + b * t.y;
    v[8 + j] = DIR > 0 ? b * t.x + a * t.y : b * t.x - a * t.y;
  }
}

// The turn of elements 16 l + j.  The other halves come from `mine`, the wave's own piece of LDS: [16][64 lanes], no barrier.
template <bool IL, int DIR>
__device__ __forceinline__ void turn_elements(float (&v)[16], float* mine, const float2* cs, const RotParams& p, int l) {
  const int np = p.rot >> 1, lane = threadIdx.x & 63, e0 = 16 * l;
  float other[16];
  if constexpr (IL) {
#pragma unroll
    for (int j = 0; j < 16; ++j) other[j] = v[j ^ 1];
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) mine[j * 64 + lane] = v[j];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int e = e0 + j, o = e < np ? e + np : e < p.rot ? e - np : e;
      other[j] = mine[(o & 15) * 64 + lane - l + (o >> 4)];
    }
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int e = e0 + j;
    if (e < p.rot) {
      const float2 t = cs[IL ? e >> 1 : e < np ? e : e - np];
      const bool first = IL ? !(j & 1) : e < np;
      v[j] = v[j] * t.x + (first == (DIR > 0) ? -other[j] : other[j]) * t.y;
    }
  }
}

// item e of a group: token and head (rows and heads are addressed from the group's first token)
struct Item { int t, head; bool on; };
__device__ __forceinline__ Item item_of(const RotParams& p, const Side& s, int e, int n, int lanes, int lshift) {
  Item it;
  it.t = s.width == 1 ? e : (int)__umulhi((uint32_t)e, s.magic);
  const int hl = e - it.t * s.width;
  it.head = hl >> lshift;
  it.on = e < n && (hl & (p.lph - 1)) < lanes;
  return it;
}

template <typename T, bool NORM, bool IL, Deal DEAL>
__global__ __launch_bounds__(256) void qk_rotary_kernel(RotParams p) {
  typedef Own<T, IL, DEAL> O;
  __shared__ float2 cs[ANGLES];
  __shared__ float other[O::ELEM && !IL ? 4 * 1024 : 1];
  float* mine = other + (O::ELEM && !IL ? (threadIdx.x >> 6) * 1024 : 0);
  const bool keys = (int)blockIdx.x >= p.side[0].blocks;
  const Side s = p.side[keys];
  const int blk = (int)blockIdx.x - (keys ? p.side[0].blocks : 0);
  const int np = p.rot >> 1, nrl = (np + 7) >> 3, lanes = O::lanes(p);
  const int lshift = __ffs(p.lph) - 1;
  const int l = threadIdx.x & (p.lph - 1);     // the same for every item of the thread: width and 256 are multiples of lph
  const bool rotates = l < nrl;
  const int valid = max(0, min(8, np - 8 * l));
  float gm[16];
  if (NORM) O::load_row(gm, s.gamma, p, min(l, lanes - 1), min(l, lanes - 1) < nrl);
  const float inv_d = 1.f / (float)p.d;
  for (int64_t grp = blk; grp < s.groups; grp += s.blocks) {
    const int64_t t0 = grp * s.tb;
    const int nt = (int)min((int64_t)s.tb, p.T - t0), n = nt * s.width;
    const T* x = (const T*)s.x + t0 * s.ldx;
    T* out = (T*)s.out + t0 * s.ldo;
    for (int e0 = 0; e0 < n; e0 += 256) {
      const Item it = item_of(p, s, e0 + threadIdx.x, n, lanes, lshift);
      typename O::Raw raw;
      O::load(raw, x + it.t * s.ldx + it.head * p.d, p, l, it.on);
      if (e0 == 0) {   // the first load is in flight meanwhile
        __syncthreads();
        group_angles(cs, p, t0, nt);
        __syncthreads();
      }
      float v[16];
      O::unpack(v, raw, rotates);
      if (NORM) {
        float ss = 0.f;
        if (it.on) {
#pragma unroll
          for (int j = 0; j < 16; ++j) ss += v[j] * (v[j] * inv_d);   // (the mean, not the sum, has to stay in range)
        }
        const float rstd = 1.f / sqrtf(head_sum(ss, p.lph) + p.eps);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = v[j] * rstd * gm[j];
      }
      if (it.on) {
        if constexpr (O::ELEM) turn_elements<IL, 1>(v, mine, cs + it.t * np, p, l);
        else if (rotates) turn<1>(v, cs + it.t * np + 8 * l, O::VEC ? 8 : valid);
        O::store(out + it.t * s.ldo + it.head * p.d, v, p, l, rotates);
      }
    }
  }
}

// Backward of norm and rotation.  dgamma: every thread sums its own elements of the head over the items it meets, then
// lanes with the same elements, the waves and (second kernel) the blocks are added in a fixed order: no atomics, results
// do not change from run to run.
// Waves per SIMD: halves of pairs fetched through LDS need 164 registers (8629 rows of 24 fp32 heads of 128, forward and
// backward: with four waves and 39 registers spilled 191 us, with three 141); element by element four are better (6896 rows
// of 24 bf16 heads of 80, 40 of them turned: 58 us, with three 65).
template <typename T, bool IL, Deal DEAL>
__global__ __launch_bounds__(256, DEAL == ELEMENTS && !IL ? 3 : 4) void qk_norm_rotary_bwd_kernel(RotParams p) {
  typedef Own<T, IL, DEAL> O;
  __shared__ float2 cs[ANGLES];
  __shared__ float red[4][MAX_D];
  __shared__ float other[O::ELEM && !IL ? 4 * 1024 : 1];
  float* mine = other + (O::ELEM && !IL ? (threadIdx.x >> 6) * 1024 : 0);
  const bool keys = (int)blockIdx.x >= p.side[0].blocks;
  const Side s = p.side[keys];
  const int blk = (int)blockIdx.x - (keys ? p.side[0].blocks : 0);
  const int np = p.rot >> 1, nrl = (np + 7) >> 3, lanes = O::lanes(p);
  const int lshift = __ffs(p.lph) - 1;
  const int l = threadIdx.x & (p.lph - 1);
  const bool rotates = l < nrl;
  const int valid = max(0, min(8, np - 8 * l));
  float gm[16], acc[16];
  O::load_row(gm, s.gamma, p, min(l, lanes - 1), min(l, lanes - 1) < nrl);
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[j] = 0.f;
  const float inv_d = 1.f / (float)p.d;
  for (int64_t grp = blk; grp < s.groups; grp += s.blocks) {
    const int64_t t0 = grp * s.tb;
    const int nt = (int)min((int64_t)s.tb, p.T - t0), n = nt * s.width;
    const T* x = (const T*)s.x + t0 * s.ldx;
    const T* dy = (const T*)s.dy + t0 * s.lddy;
    T* out = (T*)s.out + t0 * s.ldo;
    for (int e0 = 0; e0 < n; e0 += 256) {
      const Item it = item_of(p, s, e0 + threadIdx.x, n, lanes, lshift);
      typename O::Raw rx, rd;
      O::load(rx, x + it.t * s.ldx + it.head * p.d, p, l, it.on);
      O::load(rd, dy + it.t * s.lddy + it.head * p.d, p, l, it.on);
      if (e0 == 0) {
        __syncthreads();
        group_angles(cs, p, t0, nt);
        __syncthreads();
      }
      float v[16], g[16];
      O::unpack(v, rx, rotates);
      O::unpack(g, rd, rotates);
      float ss = 0.f, sg = 0.f;
      if (it.on) {
        if constexpr (O::ELEM) turn_elements<IL, -1>(g, mine, cs + it.t * np, p, l);
        else if (rotates) turn<-1>(g, cs + it.t * np + 8 * l, O::VEC ? 8 : valid);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          ss += v[j] * (v[j] * inv_d);
          sg += g[j] * gm[j] * v[j];
        }
      }
      const float rstd = 1.f / sqrtf(head_sum(ss, p.lph) + p.eps);
      const float mean = head_sum(sg, p.lph) * rstd * inv_d;   // mean(g gamma xhat)
      if (it.on) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float xhat = v[j] * rstd;
          acc[j] += g[j] * xhat;
          g[j] = rstd * (g[j] * gm[j] - xhat * mean);
        }
        O::store(out + it.t * s.ldo + it.head * p.d, g, p, l, rotates);
      }
    }
  }
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    for (int o = 32; o >= p.lph; o >>= 1) acc[j] += __shfl_xor(acc[j], o, 64);
  if (lane < p.lph && l < lanes) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {   // (sums are in pair order whatever the storage order)
      const int i = O::index(p, l, j);
      if (i >= 0) red[wave][i] = acc[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.d; i += 256)
    s.partial[(int64_t)blk * p.d + i] = red[0][i] + red[1][i] + red[2][i] + red[3][i];
}

// dgamma[c] = sum over blocks of partial[block][c]: a block adds 16 columns, 64 runs of partial rows side by side
__global__ __launch_bounds__(1024) void dgamma_sum_kernel(const float* __restrict__ part_q, const float* __restrict__ part_k,
                                                          float* __restrict__ dgq, float* __restrict__ dgk, int blocks_q,
                                                          int blocks_k, int d) {
  __shared__ float red[64][17];
  const float* part = blockIdx.y ? part_k : part_q;
  const int blocks = blockIdx.y ? blocks_k : blocks_q;
  const int c = threadIdx.x & 15, run = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float a = 0.f;
  if (col < d) {
#pragma unroll 8
    for (int b = run; b < blocks; b += 64) a += part[(int64_t)b * d + col];
  }
  red[run][c] = a;
  __syncthreads();
  if (run < 8) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += red[8 * run + i][c];
    red[8 * run][c] = v;
  }
  __syncthreads();
  if (run == 0 && col < d) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += red[8 * i][c];
    (blockIdx.y ? dgk : dgq)[col] = v;
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Lanes per head, tokens per group and blocks of each side; `most`: blocks of both sides.
void plan(RotParams& p, Deal deal, int n_head, int n_kv, int rounds, int64_t most) {
  const int np = p.rot / 2, lanes = deal == ELEMENTS ? (p.d + 15) / 16 : (np + 7) / 8 + (p.d - p.rot + 15) / 16;
  p.lph = 1;
  while (p.lph < lanes) p.lph *= 2;
  for (int i = 0; i < 2; ++i) {
    Side& s = p.side[i];
    s.heads = i ? n_kv : n_head;
    s.width = std::max(1, s.heads * p.lph);
    // A group is what a block has between two barriers: `rounds` items of each thread, fewer where the rows would not
    // give every CU two blocks (640 rows of 8 heads: 80 blocks of 8 rows a side instead of 10 of 64).
    int64_t tb = std::max<int64_t>(1, 256 * rounds / s.width);
    tb = std::min<int64_t>(tb, std::max<int64_t>(std::max(1, 256 / s.width), p.T / (2 * sk_num_cus())));
    if (np) tb = std::min<int64_t>(tb, ANGLES / np);
    s.tb = (int)tb;
    s.groups = s.heads ? (p.T + tb - 1) / tb : 0;
    s.magic = (uint32_t)((0x100000000ull + s.width - 1) / s.width);
    const int64_t share = std::max<int64_t>(1, most * s.heads / (n_head + n_kv));
    s.blocks = (int)std::min<int64_t>(s.groups, share);
  }
}

template <typename T, bool NORM, bool IL>
void launch_fwd(const RotParams& p, Deal deal, hipStream_t stream) {
  const dim3 grid((unsigned)(p.side[0].blocks + p.side[1].blocks));
  if (deal == PAIRS) hipLaunchKernelGGL((qk_rotary_kernel<T, NORM, IL, PAIRS>), grid, dim3(256), 0, stream, p);
  else if (deal == ELEMENTS) hipLaunchKernelGGL((qk_rotary_kernel<T, NORM, IL, ELEMENTS>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((qk_rotary_kernel<T, NORM, IL, SCALARS>), grid, dim3(256), 0, stream, p);
}
template <typename T>
void launch_fwd(const RotParams& p, bool norm, bool il, Deal deal, hipStream_t stream) {
  if (norm && il) launch_fwd<T, true, true>(p, deal, stream);
  else if (norm) launch_fwd<T, true, false>(p, deal, stream);
  else if (il) launch_fwd<T, false, true>(p, deal, stream);
  else launch_fwd<T, false, false>(p, deal, stream);
}

template <typename T, bool IL>
void launch_bwd(const RotParams& p, Deal deal, hipStream_t stream) {
  const dim3 grid((unsigned)(p.side[0].blocks + p.side[1].blocks));
  if (deal == PAIRS) hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<T, IL, PAIRS>), grid, dim3(256), 0, stream, p);
  else if (deal == ELEMENTS) hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<T, IL, ELEMENTS>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((qk_norm_rotary_bwd_kernel<T, IL, SCALARS>), grid, dim3(256), 0, stream, p);
}
template <typename T>
void launch_bwd(const RotParams& p, bool il, Deal deal, hipStream_t stream) {
  if (il) launch_bwd<T, true>(p, deal, stream);
  else launch_bwd<T, false>(p, deal, stream);
}

Deal deal_of(bool rows16, int d, int rot) {
  return !rows16 || d % 8 ? SCALARS : d % 16 == 0 && rot % 16 == 0 ? PAIRS : ELEMENTS;
}

int check_shape(const char* who, const int64_t* pos, const uint64_t* turns, int64_t T, int n_head, int n_kv, int d, int rot,
                int dtype) {
  SK_CHECK_ARG(dtype == SK_F32 || dtype == SK_BF16, "%s: bad dtype %d", who, dtype);
  SK_CHECK_ARG(T >= 0 && n_head > 0 && n_kv >= 0 && n_head <= 512 && n_kv <= 512, "%s: bad shape (T %lld, heads %d and %d)",
               who, (long long)T, n_head, n_kv);
  SK_CHECK_ARG(d > 0 && d <= MAX_D, "%s: head size %d must be in 1..%d", who, d, MAX_D);
  SK_CHECK_ARG(rot >= 0 && rot % 2 == 0 && rot <= d, "%s: rotated part %d must be even and at most the head size %d", who, rot, d);
  SK_CHECK_ARG(T == 0 || rot == 0 || (pos && turns), "%s: null pointer", who);
  return SK_OK;
}

}  // namespace

extern "C" int64_t skhip_qk_norm_rotary_bwd_ws_floats(int d) { return d > 0 && d <= MAX_D ? (int64_t)(BWD_BLOCKS + 1) * d : 0; }

extern "C" int skhip_qk_rotary(const void* q, const void* k, void* q_out, void* k_out, const int64_t* pos,
                               const uint64_t* turns, float amplitude, const float* gamma_q, const float* gamma_k, float eps,
                               int64_t T, int n_head, int n_kv, int d, int rot, int64_t ldq, int64_t ldk, int64_t ldq_out,
                               int64_t ldk_out, int interleaved, int inverse, int dtype, void* stream_) {
  const char* who = "skhip_qk_rotary";
  hipStream_t stream = (hipStream_t)stream_;
  int rc = check_shape(who, pos, turns, T, n_head, n_kv, d, rot, dtype);
  if (rc) return rc;
  if (T == 0) return SK_OK;
  SK_CHECK_ARG(q && q_out && (n_kv == 0 || (k && k_out)), "%s: null pointer", who);
  SK_CHECK_ARG(!gamma_q || n_kv == 0 || gamma_k, "%s: one norm weight without the other", who);
  SK_CHECK_ARG(!(gamma_q && inverse), "%s: the inverse turn takes no norm", who);
  SK_CHECK_ARG(ldq >= (int64_t)n_head * d && ldq_out >= (int64_t)n_head * d && (n_kv == 0 ||
               (ldk >= (int64_t)n_kv * d && ldk_out >= (int64_t)n_kv * d)), "%s: row stride below the row's length", who);
  RotParams p = {};
  p.pos = pos; p.turns = turns; p.amp = amplitude; p.eps = eps; p.T = T; p.d = d; p.rot = rot; p.sign = inverse ? -1 : 1;
  p.side[0].x = q; p.side[0].out = q_out; p.side[0].ldx = ldq; p.side[0].ldo = ldq_out; p.side[0].gamma = gamma_q;
  p.side[1].x = k; p.side[1].out = k_out; p.side[1].ldx = ldk; p.side[1].ldo = ldk_out; p.side[1].gamma = gamma_k;
  const int64_t per = dtype == SK_BF16 ? 8 : 4;
  bool vec = aligned16(q) && aligned16(q_out) && (ldq | ldq_out) % per == 0;
  if (n_kv) vec = vec && aligned16(k) && aligned16(k_out) && (ldk | ldk_out) % per == 0;
  const Deal deal = deal_of(vec, d, rot);
  plan(p, deal, n_head, n_kv, gamma_q ? 2 : 1, (int64_t)sk_num_cus() * 64);
  if (dtype == SK_BF16) launch_fwd<bf16_t>(p, gamma_q, interleaved, deal, stream);
  else launch_fwd<float>(p, gamma_q, interleaved, deal, stream);
  SK_CHECK_LAUNCH(who);
  return SK_OK;
}

extern "C" int skhip_qk_norm_rotary_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, void* dq,
                                        void* dk, float* dgamma_q, float* dgamma_k, const int64_t* pos,
                                        const uint64_t* turns, float amplitude, const float* gamma_q, const float* gamma_k,
                                        float eps, int64_t T, int n_head, int n_kv, int d, int rot, int64_t ldq, int64_t ldk,
                                        int64_t lddq_out, int64_t lddk_out, int64_t lddq, int64_t lddk, int interleaved,
                                        float* workspace, int64_t workspace_floats, int dtype, void* stream_) {
  const char* who = "skhip_qk_norm_rotary_bwd";
  hipStream_t stream = (hipStream_t)stream_;
  int rc = check_shape(who, pos, turns, T, n_head, n_kv, d, rot, dtype);
  if (rc) return rc;
  SK_CHECK_ARG(gamma_q && dgamma_q && (n_kv == 0 || (gamma_k && dgamma_k)), "%s: null pointer", who);
  SK_CHECK_ARG(T == 0 || (q && dq_out && dq && (n_kv == 0 || (k && dk_out && dk))), "%s: null pointer", who);
  const int64_t nq = (int64_t)n_head * d, nk = (int64_t)n_kv * d;
  SK_CHECK_ARG(T == 0 || (ldq >= nq && lddq_out >= nq && lddq >= nq && ldk >= nk && lddk_out >= nk && lddk >= nk),
               "%s: row stride below the row's length", who);
  RotParams p = {};
  p.pos = pos; p.turns = turns; p.amp = amplitude; p.eps = eps; p.T = T; p.d = d; p.rot = rot; p.sign = 1;
  Side &sq = p.side[0], &sk = p.side[1];
  sq.x = q; sq.dy = dq_out; sq.out = dq; sq.ldx = ldq; sq.lddy = lddq_out; sq.ldo = lddq; sq.gamma = gamma_q;
  sk.x = k; sk.dy = dk_out; sk.out = dk; sk.ldx = ldk; sk.lddy = lddk_out; sk.ldo = lddk; sk.gamma = gamma_k;
  const int64_t per = dtype == SK_BF16 ? 8 : 4;
  bool vec = aligned16(q) && aligned16(dq_out) && aligned16(dq) && (ldq | lddq_out | lddq) % per == 0;
  if (n_kv) vec = vec && aligned16(k) && aligned16(dk_out) && aligned16(dk) && (ldk | lddk_out | lddk) % per == 0;
  const Deal deal = deal_of(vec, d, rot);
  plan(p, deal, n_head, n_kv, 2, BWD_BLOCKS);
  const int64_t need = (int64_t)(sq.blocks + sk.blocks) * d;
  if (need > 0 && (!workspace || workspace_floats < need)) {
    sk_set_error("%s: workspace of %lld floats needed", who, (long long)need);
    return SK_ERR_WORKSPACE;
  }
  sq.partial = workspace;
  sk.partial = workspace + (int64_t)sq.blocks * d;
  if (T > 0) {
    if (dtype == SK_BF16) launch_bwd<bf16_t>(p, interleaved, deal, stream);
    else launch_bwd<float>(p, interleaved, deal, stream);
    SK_CHECK_LAUNCH(who);
  }
  hipLaunchKernelGGL(dgamma_sum_kernel, dim3((d + 15) / 16, n_kv ? 2 : 1), dim3(1024), 0, stream, sq.partial, sk.partial, dgamma_q,
                     dgamma_k, sq.blocks, sk.blocks, d);
  SK_CHECK_LAUNCH(who);
  return SK_OK;
}
