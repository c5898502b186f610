// One query per sequence against a cache of keys and values: the decoding step of the windowed attention
// (window_attn.h), with the append of the newest key and value.
//
// A sequence of n positions (the newest included) sees the first min(sinks, n) and the last min(window, n).  Position j
// lives in cache slot  j < sinks ? j : sinks + (j - sinks) % (cap - sinks):  with cap >= n that is slot j, with
// cap = sinks + window a ring that holds exactly what can still be seen, however long the text gets.
//
// Bound by HBM: the visible keys and values are read once (256 sequences x 2052 slots, 32 / 8 heads of 128 in bf16: 375 us,
// 5.5 TB/s; 64 x 4100 slots, 8 fp32 heads of 64: 198 us, 5.4).  With few sequences a block per (sequence, head) would leave
// most CUs idle, so the visible positions are cut into splits, each block leaves the running maximum, sum and weighted
// value of its part in the workspace, and a second small kernel joins them (2 sequences of 16388 visible positions, 32 / 4
// heads of 128, 67 MB: uncut 8 blocks, in splits 16.2 + 4.1 us).
//
// Heads of whole 16-byte pieces run on the matrix cores: the query heads that share a key head are the 16 columns of every
// product, so keys and values are read once for all of them.  Other rows take one block per query head on the vector ALU.
#include "window_attn.h"
#include <algorithm>

namespace {

constexpr int MAXD = 128;
constexpr int KT = 64;   // keys per pass of a wave: one per lane
constexpr int MAX_SPLITS = 512;

struct StepParams {
  const void *q, *kn, *vn;
  void *kc, *vc, *out;
  const int32_t* len;
  float* part;              // [R][H][splits][d + 2]: weighted values, maximum, sum
  int64_t ldq, ldn, ldo, ks, kp, vs, vp;   // strides: sequence (s) and position (p) of the caches
  int R, H, G, d, cap, window, sinks, splits;
  float scale;
};

// The visible positions of a sequence in order: sinks, then the window.
struct Visible {
  int n, ns, lo, count;
  __device__ __forceinline__ explicit Visible(const StepParams& p, int r) {
    n = max(0, p.len[r]);
    lo = max(0, n - p.window);
    ns = min(p.sinks, lo);
    count = ns + (n - lo);
  }
  // Positions of a split: the sequence's own, shared out evenly, `unit` at a time and four units at least, so that a short
  // sequence in a batch planned for long ones is spread as widely.
  __device__ __forceinline__ int per_split(const StepParams& p, int unit) const {
    return max(4 * unit, (count + p.splits * unit - 1) / (p.splits * unit) * unit);
  }
  __device__ __forceinline__ int pos(int u) const { return u < ns ? u : lo + (u - ns); }
  __device__ __forceinline__ int slot(const StepParams& p, int j) const {
    return j < p.sinks ? j : p.sinks + (int)((uint32_t)(j - p.sinks) % (uint32_t)(p.cap - p.sinks));
  }
};

template <typename T>
__global__ __launch_bounds__(256) void step_kernel(StepParams p, int vec) {
  __shared__ __attribute__((aligned(16))) float qs[MAXD];
  __shared__ float s_m[4], s_l[4], s_o[4][MAXD];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = blockIdx.z, h = blockIdx.y, rep = p.H / p.G, kh = h / rep, split = blockIdx.x;
  const Visible vis(p, r);
  for (int c = threadIdx.x; c < p.d; c += 256) qs[c] = Cvt<T>::to_f32(((const T*)p.q)[r * p.ldq + (int64_t)h * p.d + c]) * p.scale;
  __syncthreads();
  T* K = (T*)p.kc + r * p.ks + (int64_t)kh * p.d;
  T* V = (T*)p.vc + r * p.vs + (int64_t)kh * p.d;
  const T* kn = p.kn ? (const T*)p.kn + r * p.ldn + (int64_t)kh * p.d : nullptr;
  const T* vn = p.vn ? (const T*)p.vn + r * p.ldn + (int64_t)kh * p.d : nullptr;
  const bool writer = h % rep == 0;
  float m = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
  const int per = vis.per_split(p, KT), u_end = min(vis.count, (split + 1) * per);
  for (int u0 = split * per + wave * KT; u0 < u_end; u0 += 4 * KT) {
    const int u = u0 + lane;
    const bool on = u < u_end;
    int64_t row = 0;
    bool fresh = false;
    float s = -INFINITY;
    if (on) {
      const int j = vis.pos(u);
      row = vis.slot(p, j);
      fresh = kn && j == vis.n - 1;
      const T* kr = fresh ? kn : K + row * p.kp;
      float acc = 0.f;
      if (vec) {
        constexpr int VN = Vec16<T>::N;
        for (int c = 0; c < p.d; c += VN) {
          Vec16<T> w;
          w.v = *(const decltype(w.v)*)(kr + c);
          if (fresh && writer) *(decltype(w.v)*)(K + row * p.kp + c) = w.v;
#pragma unroll
          for (int e = 0; e < VN; ++e) acc += qs[c + e] * w.get(e);
        }
      } else {
        for (int c = 0; c < p.d; ++c) {
          if (fresh && writer) K[row * p.kp + c] = kr[c];
          acc += qs[c] * Cvt<T>::to_f32(kr[c]);
        }
      }
      s = acc;
    }
    const float mn = fmaxf(m, wave_max(s)), base = mn == -INFINITY ? 0.f : mn;   // (-inf: no score above -inf so far, or NaN scores only)
    const float alpha = m == -INFINITY ? 0.f : expf(m - mn), pr = on ? expf(s - base) : 0.f;
    l = l * alpha + wave_sum(pr);
    m = mn;
    a0 *= alpha;
    a1 *= alpha;
    const int cnt = min(KT, u_end - u0);
#pragma unroll 4
    for (int t = 0; t < cnt; ++t) {
      const float w = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(pr), t));
      const int64_t at = __builtin_amdgcn_readlane((int)row, t);   // (slots are below 2^30)
      const bool fr = __builtin_amdgcn_readlane((int)fresh, t);
      const T* vr = fr ? vn : V + at * p.vp;
      if (lane < p.d) {
        const T x = vr[lane];
        a0 += w * Cvt<T>::to_f32(x);
        if (fr && writer) V[at * p.vp + lane] = x;
      }
      if (lane + 64 < p.d) {
        const T x = vr[lane + 64];
        a1 += w * Cvt<T>::to_f32(x);
        if (fr && writer) V[at * p.vp + lane + 64] = x;
      }
    }
  }
  if (lane == 0) { s_m[wave] = m; s_l[wave] = l; }
  if (lane < p.d) s_o[wave][lane] = a0;
  if (lane + 64 < p.d) s_o[wave][lane + 64] = a1;
  __syncthreads();
  const float mm = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float f[4], ll = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = s_m[w] == -INFINITY ? (s_l[w] == 0.f ? 0.f : 1.f) : expf(s_m[w] - mm);   // (a sum of NaN scores has no maximum)
    ll += f[w] * s_l[w];
  }
  float* part = p.part + (((int64_t)r * p.H + h) * p.splits + split) * (p.d + 2);
  for (int c = threadIdx.x; c < p.d; c += 256) {
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) o += f[w] * s_o[w][c];
    if (p.splits == 1) ((T*)p.out)[r * p.ldo + (int64_t)h * p.d + c] = Cvt<T>::from_f32(ll == 0.f ? 0.f : o / ll);
    else part[c] = o;
  }
  if (p.splits > 1 && threadIdx.x == 0) { part[p.d] = mm; part[p.d + 1] = ll; }
}

// ------------------------------------------------------------------------------ matrix cores
typedef __attribute__((address_space(1))) void* gbl_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr int HEADS = 16;   // query heads per block

// byte address of 16-byte piece `piece` of row `row` of a tile whose rows are `bytes` long: pieces exchanged with the row,
// so that reads by columns spread over the banks
__device__ __forceinline__ int at(int bytes, int row, int piece) { return row * bytes + ((piece ^ (row & 7)) << 4); }

// A pass of a wave: MT positions.  Products are D[rho][c] = sum_k X[rho][k] Y[c][k] with the query head on c = lane & 15
// and g = lane / 16; scores = keys x queries, piece t holding positions 16 t + 4 g + r in register r; output = values x
// probabilities, for which the scores' registers are the Y operand as they stand.
template <typename T, int D> struct Pass;

template <int D> struct Pass<bf16_t, D> {   // v_mfma_f32_16x16x32_bf16
  static constexpr int MT = 32, PIECES = 2, NK = D / 32;
  typedef bf16x8_t frag;
  static __device__ __forceinline__ int first(int s, int g) { return 32 * s + 8 * g; }
  static __device__ __forceinline__ uint32_t sign() { return 0x80008000u; }
  static __device__ __forceinline__ f32x4_t scores(const frag (&k)[NK], const frag (&q)[NK]) {
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NK; ++s) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[s], q[s], a, 0, 0, 0);
    return a;
  }
  // o[x] (columns 16 x + 4 g + r) = alpha o[x] + values x probabilities.  The probabilities are rounded to bf16: half a
  // step of 2^-8 each, as the output's own rounding.
  static __device__ __forceinline__ void add(f32x4_t (&o)[D / 16], float alpha, const f32x4_t (&p)[PIECES], const char* v, int c, int g) {
    bf16x8_t y;
#pragma unroll
    for (int e = 0; e < 4; ++e) { y[e] = (__bf16)p[0][e]; y[4 + e] = (__bf16)p[1][e]; }
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
      typedef __attribute__((address_space(3))) s16x4_t* lds_v4;
      const int row = 4 * g + (c >> 2), col = 16 * x + 4 * (c & 3);
      s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(v + at(2 * D, row, col >> 3) + (col & 7) * 2));
      s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(v + at(2 * D, row + 16, col >> 3) + (col & 7) * 2));
      s16x8_t f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      o[x] *= alpha;
      o[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, f), y, o[x], 0, 0, 0);
    }
  }
};

template <int D> struct Pass<float, D> {    // v_mfma_f32_16x16x4_f32
  static constexpr int MT = 16, PIECES = 1, NK = D / 16;
  typedef f32x4_t frag;
  static __device__ __forceinline__ int first(int s, int g) { return 16 * s + 4 * g; }
  static __device__ __forceinline__ uint32_t sign() { return 0x80000000u; }
  static __device__ __forceinline__ f32x4_t scores(const frag (&k)[NK], const frag (&q)[NK]) {
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) a = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][j], q[s][j], a, 0, 0, 0);
    return a;
  }
  static __device__ __forceinline__ void add(f32x4_t (&o)[D / 16], float alpha, const f32x4_t (&p)[PIECES], const char* v, int c, int g) {
#pragma unroll
    for (int x = 0; x < D / 16; ++x) o[x] *= alpha;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const float w = *(const float*)(v + at(4 * D, 4 * g + r, 4 * x + (c >> 2)) + (c & 3) * 4);
        o[x] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, p[0][r], o[x], 0, 0, 0);
      }
  }
};

// Every wave keeps two passes in flight: the next pass's keys in registers and values in its own LDS buffer, by direct
// loads, while this one is multiplied; nothing is shared between waves until the end.  Positions beyond the split read the
// pass's first one again, elements beyond the head its first piece: both are cleared before they are multiplied.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void step_mfma_kernel(StepParams p, int chunks) {
  typedef Pass<T, D> P;
  typedef typename P::frag frag;
  constexpr int MT = P::MT, NK = P::NK, PE = 16 / sizeof(T);     // elements of a 16-byte piece
  constexpr int CH = D / PE, RPI = 64 / CH, NV = MT / RPI;       // pieces per row, rows per instruction, instructions per tile
  constexpr int ROWB = D * sizeof(T), TILE = MT * ROWB, LDO = D + 4;
  constexpr int BYTES = 8 * TILE > 4 * HEADS * LDO * 4 ? 8 * TILE : 4 * HEADS * LDO * 4;
  __shared__ __attribute__((aligned(1024))) char lds[BYTES];
  __shared__ float s_m[4][HEADS], s_l[4][HEADS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int r = blockIdx.z, kh = blockIdx.y / chunks, hc = blockIdx.y - kh * chunks, split = blockIdx.x;
  const int rep = p.H / p.G, h0 = kh * rep + hc * HEADS, nh = min(HEADS, rep - hc * HEADS);
  const Visible vis(p, r);
  const int per = vis.per_split(p, MT), u_beg = split * per, u_end = min(vis.count, u_beg + per);
  T* K = (T*)p.kc + r * p.ks + (int64_t)kh * p.d;
  T* V = (T*)p.vc + r * p.vs + (int64_t)kh * p.d;
  const T* kn = p.kn ? (const T*)p.kn + r * p.ldn + (int64_t)kh * p.d : nullptr;
  const T* vn = p.vn ? (const T*)p.vn + r * p.ldn + (int64_t)kh * p.d : nullptr;
  // slots without a division per position: the window meets the ring's end at most once
  const int ring = p.cap - p.sinks, x0 = max(vis.lo, p.sinks), b0 = (x0 - p.sinks) % ring;
  auto slot = [&](int u) -> int64_t {
    const int j = vis.pos(u);
    int s = b0 + (j - x0);
    s -= s >= ring ? ring : 0;
    return j < p.sinks ? j : p.sinks + s;
  };
  frag q[NK];
#pragma unroll
  for (int s = 0; s < NK; ++s) {
    uint4 v = make_uint4(0, 0, 0, 0);
    const int e = P::first(s, g);
    if (c < nh && e < p.d) v = *(const uint4*)((const T*)p.q + r * p.ldq + (int64_t)(h0 + c) * p.d + e);
    if (p.scale < 0.f) { v.x ^= P::sign(); v.y ^= P::sign(); v.z ^= P::sign(); v.w ^= P::sign(); }   // (maxima are of unscaled scores)
    q[s] = __builtin_bit_cast(frag, v);
  }
  const float cs = fabsf(p.scale) * LOG2E;
  f32x4_t o[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  frag ka[P::PIECES][NK], kb[P::PIECES][NK];
  char* mine = lds + wave * 2 * TILE;
  auto fetch = [&](int u0, char* buf, frag (&k)[P::PIECES][NK]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int row = j * RPI + lane / CH, piece = (lane % CH) ^ (row & 7);
      const int u = u0 + row < u_end ? u0 + row : u0;
      const bool fresh = vn && vis.pos(u) == vis.n - 1;
      const T* src = (fresh ? vn : V + slot(u) * p.vp) + (piece * PE < p.d ? piece * PE : 0);
      __builtin_amdgcn_global_load_lds((gbl_ptr)src, (lds_ptr)(buf + j * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < P::PIECES; ++t) {
      const int u = u0 + 16 * t + c < u_end ? u0 + 16 * t + c : u0;
      const bool fresh = kn && vis.pos(u) == vis.n - 1;
      const T* src = fresh ? kn : K + slot(u) * p.kp;
#pragma unroll
      for (int s = 0; s < NK; ++s) k[t][s] = *(const frag*)(src + (P::first(s, g) < p.d ? P::first(s, g) : 0));
    }
  };
  // one pass from registers `k` and buffer `vt`, while the next one is fetched into the others
  auto pass = [&](int u0, frag (&k)[P::PIECES][NK], frag (&next)[P::PIECES][NK], char* vt, char* vnext) {
    if (u0 + 4 * MT < u_end) {
      fetch(u0 + 4 * MT, vnext, next);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NV + P::PIECES * NK) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if (p.d < D) {               // (pieces beyond the head: an infinity there must not meet the query's zeros,
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int t = 0; t < P::PIECES; ++t) k[t][s] = P::first(s, g) < p.d ? k[t][s] : frag{};
    }
    if (u0 + MT > u_end) {       // nor one in the values read again the probabilities' zeros)
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (u0 + j * RPI + lane / CH >= u_end) *(uint4*)(vt + j * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
    }
    f32x4_t sc[P::PIECES];
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < P::PIECES; ++t) {
      sc[t] = P::scores(k[t], q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (u0 + 16 * t + 4 * g + e >= u_end) sc[t][e] = -INFINITY;
        mx = fmaxf(mx, sc[t][e]);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx), mc = mn == -INFINITY ? 0.f : mn * cs;
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(fmaf(m, cs, -mc));
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < P::PIECES; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[t][e] = __builtin_amdgcn_exp2f(fmaf(sc[t][e], cs, -mc));
        sum += sc[t][e];
      }
    l = l * alpha + sum;      // (of this lane's positions; the four lanes of a head are added at the end)
    P::add(o, alpha, sc, vt, c, g);
  };
  const int first = u_beg + wave * MT;
  if (first < u_end) fetch(first, mine, ka);
  for (int u0 = first; u0 < u_end; u0 += 8 * MT) {   // (two passes a round: no register moves, which would wait for the loads)
    pass(u0, ka, kb, mine, mine + TILE);
    if (u0 + 4 * MT < u_end) pass(u0 + 4 * MT, kb, ka, mine + TILE, mine);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the newest key and value go into their slot (every reader took them from the new rows)
  if (kn && hc == 0 && vis.count > 0 && u_beg < vis.count && u_end == vis.count) {
    const int64_t at_slot = slot(vis.count - 1);
    const int n = p.d / PE;
    for (int e = threadIdx.x; e < 2 * n; e += 256) {   // keys, then values
      const bool isv = e >= n;
      const int x = PE * (isv ? e - n : e);
      *(uint4*)((isv ? V + at_slot * p.vp : K + at_slot * p.kp) + x) = *(const uint4*)((isv ? vn : kn) + x);
    }
  }
  // the block's waves joined through LDS
  __syncthreads();
  float* so = (float*)lds;   // [4][HEADS][LDO]
  if (c < nh) {
#pragma unroll
    for (int x = 0; x < D / 16; ++x) *(float4*)&so[(wave * HEADS + c) * LDO + 16 * x + 4 * g] = make_float4(o[x][0], o[x][1], o[x][2], o[x][3]);
    if (g == 0) { s_m[wave][c] = m; s_l[wave][c] = l; }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nh * (D / 4); e += 256) {
    const int hh = e / (D / 4), x = 4 * (e - hh * (D / 4));
    if (x >= p.d) continue;
    const float mm = fmaxf(fmaxf(s_m[0][hh], s_m[1][hh]), fmaxf(s_m[2][hh], s_m[3][hh]));
    float ll = 0.f, a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = s_m[w][hh] == -INFINITY ? (s_l[w][hh] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f((s_m[w][hh] - mm) * cs);
      const float4 v = *(const float4*)&so[(w * HEADS + hh) * LDO + x];
      ll += f * s_l[w][hh];
      a[0] += f * v.x; a[1] += f * v.y; a[2] += f * v.z; a[3] += f * v.w;
    }
    if (p.splits == 1) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      T* out = (T*)p.out + r * p.ldo + (int64_t)(h0 + hh) * p.d + x;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = Cvt<T>::from_f32(a[i] * inv);
    } else {
      float* part = p.part + (((int64_t)r * p.H + h0 + hh) * p.splits + split) * (p.d + 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) part[x + i] = a[i];
      if (x == 0) { part[p.d] = mm * cs * (1.f / LOG2E); part[p.d + 1] = ll; }
    }
  }
}

// One block per (sequence, head), 512 threads: a thread adds one column over every fourth split.  The columns of the first
// 64 splits are on their way with the splits' maxima and sums: one trip to memory for most launches.
template <typename T>
__global__ __launch_bounds__(512) void step_join_kernel(StepParams p) {
  __shared__ float s_m[MAX_SPLITS], s_l[MAX_SPLITS], red[4][MAXD];
  const int64_t rh = blockIdx.x;
  const int r = (int)(rh / p.H), h = (int)(rh - (int64_t)r * p.H), lane = threadIdx.x & 63;
  const float* part = p.part + rh * p.splits * (p.d + 2);
  const int col = threadIdx.x & (MAXD - 1), run = threadIdx.x / MAXD;
  constexpr int FIRST = 16;
  float v[FIRST];
#pragma unroll
  for (int i = 0; i < FIRST; ++i) {
    const int s = run + 4 * i;
    v[i] = col < p.d && s < p.splits ? part[(int64_t)s * (p.d + 2) + col] : 0.f;
  }
  for (int s = threadIdx.x; s < p.splits; s += 512) {
    s_m[s] = part[(int64_t)s * (p.d + 2) + p.d];
    s_l[s] = part[(int64_t)s * (p.d + 2) + p.d + 1];
  }
  __syncthreads();
  float m = -INFINITY, l = 0.f;   // every wave for itself
  for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, s_m[s]);
  m = wave_max(m);
  for (int s = lane; s < p.splits; s += 64) l += s_m[s] == -INFINITY ? s_l[s] : expf(s_m[s] - m) * s_l[s];   // (0 or NaN)
  l = wave_sum(l);
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < FIRST; ++i) {
    const int s = run + 4 * i;
    if (s < p.splits && s_m[s] != -INFINITY) a += expf(s_m[s] - m) * v[i];
  }
  if (col < p.d) {
#pragma unroll 8
    for (int s = run + 4 * FIRST; s < p.splits; s += 4)
      a += s_m[s] == -INFINITY ? 0.f : expf(s_m[s] - m) * part[(int64_t)s * (p.d + 2) + col];
  }
  red[run][col] = a;
  __syncthreads();
  if (run == 0 && col < p.d)
    ((T*)p.out)[r * p.ldo + (int64_t)h * p.d + col] =
        Cvt<T>::from_f32(l == 0.f ? 0.f : (red[0][col] + red[1][col] + red[2][col] + red[3][col]) / l);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Splits: enough blocks to give every CU two, each with at least one pass of its four waves.  Blocks that do not fall evenly
// on the CUs leave some idle while others have one more to do; then more splits, up to eight blocks a CU and not under four
// passes each, until nine tenths are in use: 70 sequences of 8 heads of 64 over a window of 8192 take 302 us as 560 blocks,
// 229 (5.1 TB/s) as 2240; 40 of them 178 and 136.  Ragged lengths are uneven either way: 300 sequences of one head, 100 to
// 9000 positions, window 2048: 62 and 66.
void plan(StepParams& p, bool mfma, int dtype) {
  const int64_t most = std::min<int64_t>((int64_t)p.window + p.sinks, p.cap), unit = !mfma ? KT : dtype == SK_BF16 ? 32 : 16;   // positions a wave takes at a time
  const int64_t blocks = (int64_t)p.R * (mfma ? p.G * ((p.H / p.G + HEADS - 1) / HEADS) : p.H), cus = sk_num_cus();
  const int64_t units = (most + unit - 1) / unit;
  auto per = [&](int64_t s) { return (units + s - 1) / s; };
  auto uneven = [&](int64_t s) {
    const int64_t n = blocks * ((units + per(s) - 1) / per(s));
    return 10 * n < 9 * ((n + cus - 1) / cus * cus);
  };
  int64_t s = std::max<int64_t>(1, std::min({(int64_t)MAX_SPLITS, 2 * cus / std::max<int64_t>(1, blocks), units / 4}));
  if (uneven(s))
    for (int64_t t = s + 1; t <= std::min<int64_t>(MAX_SPLITS, units / 16) && t * blocks <= 8 * cus; ++t)
      if (!uneven(t)) { s = t; break; }
  p.splits = (int)((units + per(s) - 1) / per(s));
}

int64_t ws_floats(const StepParams& p) { return p.splits > 1 ? (int64_t)p.R * p.H * p.splits * (p.d + 2) : 0; }

}  // namespace

extern "C" int64_t skhip_window_attn_step_ws_floats(int R, int n_head, int n_kv, int d, int cap, int window, int sinks) {
  if (R <= 0 || n_head <= 0 || n_kv <= 0 || d <= 0 || cap <= 0 || window < 1 || sinks < 0) return 0;
  StepParams p = {};
  p.R = R; p.H = n_head; p.G = n_kv; p.d = d; p.cap = cap; p.window = window; p.sinks = sinks;
  if (n_head % n_kv) return 0;
  // the largest of the paths' needs: which one a call takes depends on its pointers and strides
  plan(p, false, SK_F32);
  int64_t n = ws_floats(p);
  plan(p, true, SK_F32);
  n = std::max(n, ws_floats(p));
  plan(p, true, SK_BF16);
  return std::max(n, ws_floats(p));
}

extern "C" int skhip_window_attn_step(const void* q, const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                                      void* out, const int32_t* kv_len, int R, int n_head, int n_kv, int d, int cap,
                                      int64_t ldq, int64_t ld_new, int64_t ldo, int64_t k_row, int64_t k_pos, int64_t v_row,
                                      int64_t v_pos, float scale, int window, int sinks, float* workspace,
                                      int64_t workspace_floats, int dtype, void* stream_) {
  const char* who = "skhip_window_attn_step";
  hipStream_t stream = (hipStream_t)stream_;
  SK_CHECK_ARG(dtype == SK_F32 || dtype == SK_BF16, "%s: bad dtype %d", who, dtype);
  SK_CHECK_ARG(R >= 0 && R <= 65535 && n_head > 0 && n_head <= 32767 && n_kv > 0 && cap <= (1 << 30), "%s: bad shape", who);
  SK_CHECK_ARG(n_head % n_kv == 0, "%s: %d query heads do not share %d key heads evenly", who, n_head, n_kv);
  SK_CHECK_ARG(d > 0 && d <= MAXD, "%s: head size %d must be in 1..%d", who, d, MAXD);
  SK_CHECK_ARG(window >= 1 && sinks >= 0 && cap > sinks && cap - sinks >= window,
               "%s: a cache of %d slots cannot hold %d sinks and a window of %d", who, cap, sinks, window);
  SK_CHECK_ARG(!k_new == !v_new, "%s: a new key without a value", who);
  if (R == 0) return SK_OK;
  SK_CHECK_ARG(q && k_cache && v_cache && out && kv_len, "%s: null pointer", who);
  const int64_t nq = (int64_t)n_head * d, nk = (int64_t)n_kv * d;
  SK_CHECK_ARG(ldq >= nq && ldo >= nq && k_pos >= nk && v_pos >= nk && (!k_new || ld_new >= nk),
               "%s: row stride below the row's length", who);
  StepParams p = {};
  p.q = q; p.kn = k_new; p.vn = v_new; p.kc = k_cache; p.vc = v_cache; p.out = out; p.len = kv_len; p.part = workspace;
  p.ldq = ldq; p.ldn = ld_new; p.ldo = ldo; p.ks = k_row; p.kp = k_pos; p.vs = v_row; p.vp = v_pos;
  p.R = R; p.H = n_head; p.G = n_kv; p.d = d; p.cap = cap; p.window = window; p.sinks = sinks; p.scale = scale;
  const int64_t strides = k_row | k_pos | v_row | v_pos | ldq | (k_new ? ld_new : 0);
  const int per = dtype == SK_BF16 ? 8 : 4;
  const bool rows16 = d % per == 0 && strides % per == 0 && aligned16(q) && aligned16(k_cache) && aligned16(v_cache) &&
                      aligned16(k_new) && aligned16(v_new);
  // (the matrix cores take maxima of unscaled scores, which a scale of 0 or inf cannot stand for)
  const bool mfma = rows16 && fabsf(scale) >= 1e-30f && scale - scale == 0.f;
  plan(p, mfma, dtype);
  if (ws_floats(p) > 0 && (!workspace || workspace_floats < ws_floats(p))) {
    sk_set_error("%s: workspace of %lld floats needed", who, (long long)ws_floats(p));
    return SK_ERR_WORKSPACE;
  }
  const int chunks = (n_head / n_kv + HEADS - 1) / HEADS;
  const dim3 grid(p.splits, mfma ? n_kv * chunks : n_head, R);
  if (dtype == SK_BF16) {
    if (mfma && d <= 64) hipLaunchKernelGGL((step_mfma_kernel<bf16_t, 64>), grid, dim3(256), 0, stream, p, chunks);
    else if (mfma) hipLaunchKernelGGL((step_mfma_kernel<bf16_t, 128>), grid, dim3(256), 0, stream, p, chunks);
    else hipLaunchKernelGGL((step_kernel<bf16_t>), grid, dim3(256), 0, stream, p, (int)rows16);
  } else {
    if (mfma && d <= 64) hipLaunchKernelGGL((step_mfma_kernel<float, 64>), grid, dim3(256), 0, stream, p, chunks);
    else if (mfma) hipLaunchKernelGGL((step_mfma_kernel<float, 128>), grid, dim3(256), 0, stream, p, chunks);
    else hipLaunchKernelGGL((step_kernel<float>), grid, dim3(256), 0, stream, p, (int)rows16);
  }
  if (p.splits > 1) {
    const dim3 join((unsigned)(R * n_head));
    if (dtype == SK_BF16) hipLaunchKernelGGL((step_join_kernel<bf16_t>), join, dim3(512), 0, stream, p);
    else hipLaunchKernelGGL((step_join_kernel<float>), join, dim3(512), 0, stream, p);
  }
  SK_CHECK_LAUNCH(who);
  return SK_OK;
}
