// One query per sequence against a cache of keys and values: the decoding step of the windowed attention
// (window_attn.h), with the append of the newest key and value.
//
// A sequence of n positions (the newest included) sees the first min(sinks, n) and the last min(window, n).  Position j
// lives in cache slot  j < sinks ? j : sinks + (j - sinks) % (cap - sinks):  with cap >= n that is slot j, with
// cap = sinks + window a ring that holds exactly what can still be seen, however long the text gets.
//
// Bound by HBM: the visible keys and values are read once.  With few sequences a block per (sequence, head) would leave
// most CUs idle, so the visible positions are cut into splits, each block leaves the running maximum, sum and weighted
// value of its part in the workspace, and a second small kernel joins them.
//
// bf16 heads of whole 16-byte pieces run on the matrix cores (v_mfma_f32_16x16x32_bf16): the query heads that share a key
// head are the 16 columns of every product, so keys and values are read once for all of them.  Other rows and fp32 take
// one block per query head on the vector ALU.
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
  int R, H, G, d, cap, window, sinks, splits, per;   // per: visible positions of a split (multiple of 4 * KT)
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
  const int u_end = min(vis.count, (split + 1) * p.per);
  for (int u0 = split * p.per + wave * KT; u0 < u_end; u0 += 4 * KT) {
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
    const float mn = fmaxf(m, wave_max(s));   // finite: the pass holds at least one position (NaN scores stay NaN)
    const float alpha = m == -INFINITY ? 0.f : expf(m - mn), pr = on ? expf(s - mn) : 0.f;
    l = l * alpha + wave_sum(pr);
    m = mn;
    a0 *= alpha;
    a1 *= alpha;
    const int cnt = min(KT, u_end - u0);
#pragma unroll 4
    for (int t = 0; t < cnt; ++t) {
      const float w = __shfl(pr, t, 64);
      const int64_t at = __shfl(row, t, 64);
      const bool fr = __shfl((int)fresh, t, 64);
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
    f[w] = s_m[w] == -INFINITY ? 0.f : expf(s_m[w] - mm);
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
constexpr int MT = 32;      // positions per pass of a wave
constexpr int HEADS = 16;   // query heads per block

__device__ __forceinline__ f32x4_t mfma16(bf16x8_t x, bf16x8_t y, f32x4_t acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0);
}
// byte address of chunk `chunk` of row `row` of a tile of D columns: chunks exchanged with the row, so that the
// transposing reads spread over the banks
template <int D> __device__ __forceinline__ int at(int row, int chunk) { return row * (2 * D) + ((chunk ^ (row & 7)) << 4); }

// Products are D[rho][c] = sum_k X[rho][k] Y[c][k] with the query head on c = lane & 15: scores = keys (straight from
// memory, a lane's 16 bytes of a row) x queries; output = values (transposed LDS read) x probabilities, which the score
// accumulators are in the order 4 g + r, 16 + 4 g + r (g = lane / 16).  Every wave keeps two passes of 32 positions in
// flight: the next pass's keys in registers and values in its own LDS buffer, by direct loads, while this one is
// multiplied; nothing is shared between waves until the end.  Positions beyond the split read its first one again and
// are masked, elements beyond the head its first piece against a zero query.
template <int D>
__global__ __launch_bounds__(256, 2) void step_mfma_kernel(StepParams p, int chunks) {
  constexpr int NS = D / 32, NV = D / 16, CH = D / 8, RPI = 64 / CH;   // k steps, value instructions, pieces per row, rows per instruction
  constexpr int TILE = MT * 2 * D, LDO = D + 4;
  __shared__ __attribute__((aligned(1024))) char lds[8 * TILE > 4 * HEADS * LDO * 4 ? 8 * TILE : 4 * HEADS * LDO * 4];
  __shared__ float s_m[4][HEADS], s_l[4][HEADS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  const int r = blockIdx.z, kh = blockIdx.y / chunks, hc = blockIdx.y - kh * chunks, split = blockIdx.x;
  const int rep = p.H / p.G, h0 = kh * rep + hc * HEADS, nh = min(HEADS, rep - hc * HEADS);
  const Visible vis(p, r);
  const int u_beg = split * p.per, u_end = min(vis.count, u_beg + p.per);
  bf16_t* K = (bf16_t*)p.kc + r * p.ks + (int64_t)kh * p.d;
  bf16_t* V = (bf16_t*)p.vc + r * p.vs + (int64_t)kh * p.d;
  const bf16_t* kn = p.kn ? (const bf16_t*)p.kn + r * p.ldn + (int64_t)kh * p.d : nullptr;
  const bf16_t* vn = p.vn ? (const bf16_t*)p.vn + r * p.ldn + (int64_t)kh * p.d : nullptr;
  // slots without a division per position: the window meets the ring's end at most once
  const int ring = p.cap - p.sinks, x0 = max(vis.lo, p.sinks), b0 = (x0 - p.sinks) % ring;
  auto slot = [&](int u) -> int64_t {
    const int j = vis.pos(u);
    int s = b0 + (j - x0);
    s -= s >= ring ? ring : 0;
    return j < p.sinks ? j : p.sinks + s;
  };
  bf16x8_t q[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    uint4 v = make_uint4(0, 0, 0, 0);
    const int e = 32 * s + 8 * g;
    if (c < nh && e < p.d) v = *(const uint4*)((const bf16_t*)p.q + r * p.ldq + (int64_t)(h0 + c) * p.d + e);
    if (p.scale < 0.f) { v.x ^= 0x80008000u; v.y ^= 0x80008000u; v.z ^= 0x80008000u; v.w ^= 0x80008000u; }
    q[s] = __builtin_bit_cast(bf16x8_t, v);
  }
  const float cs = fabsf(p.scale) * LOG2E;
  f32x4_t o[NV];
#pragma unroll
  for (int t = 0; t < NV; ++t) o[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  bf16x8_t kc[2][NS], kx[2][NS];
  char* mine = lds + wave * 2 * TILE;
  auto fetch = [&](int u0, char* buf, bf16x8_t (&k)[2][NS]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int row = j * RPI + lane / CH, piece = (lane % CH) ^ (row & 7);
      const int u = u0 + row < u_end ? u0 + row : u0;
      const bool fresh = vn && vis.pos(u) == vis.n - 1;
      const bf16_t* src = (fresh ? vn : V + slot(u) * p.vp) + (piece * 8 < p.d ? piece * 8 : 0);
      __builtin_amdgcn_global_load_lds((gbl_ptr)src, (lds_ptr)(buf + j * 1024), 16, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int u = u0 + 16 * t + c < u_end ? u0 + 16 * t + c : u0;
      const bool fresh = kn && vis.pos(u) == vis.n - 1;
      const bf16_t* src = fresh ? kn : K + slot(u) * p.kp;
#pragma unroll
      for (int s = 0; s < NS; ++s) k[t][s] = *(const bf16x8_t*)(src + (32 * s + 8 * g < p.d ? 32 * s + 8 * g : 0));
    }
  };
  // one pass from registers `k` and buffer `vt`, while the next one is fetched into the others
  auto pass = [&](int u0, bf16x8_t (&k)[2][NS], bf16x8_t (&next)[2][NS], char* vt, char* vnext) {
    if (u0 + 4 * MT < u_end) {
      fetch(u0 + 4 * MT, vnext, next);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NV + 2 * NS) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    f32x4_t sc[2];
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NS; ++s) sc[t] = mfma16(k[t][s], q[s], sc[t]);
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
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[t][e] = __builtin_amdgcn_exp2f(fmaf(sc[t][e], cs, -mc));
        sum += sc[t][e];
      }
    l = l * alpha + sum;      // (of this lane's positions; the four lanes of a head are added at the end)
    bf16x8_t y;               // probabilities rounded to bf16: half a step of 2^-8 each, as the output's own rounding
#pragma unroll
    for (int e = 0; e < 4; ++e) { y[e] = (__bf16)sc[0][e]; y[4 + e] = (__bf16)sc[1][e]; }
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      typedef __attribute__((address_space(3))) s16x4_t* lds_v4;
      const int row = 4 * g + (c >> 2), col = 16 * x + 4 * (c & 3);
      s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vt + at<D>(row, col >> 3) + (col & 7) * 2));
      s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vt + at<D>(row + 16, col >> 3) + (col & 7) * 2));
      s16x8_t f = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      o[x] *= alpha;
      o[x] = mfma16(__builtin_bit_cast(bf16x8_t, f), y, o[x]);
    }
  };
  const int first = u_beg + wave * MT;
  if (first < u_end) fetch(first, mine, kc);
  for (int u0 = first; u0 < u_end; u0 += 8 * MT) {   // (two passes a round: no register moves, which would wait for the loads)
    pass(u0, kc, kx, mine, mine + TILE);
    if (u0 + 4 * MT < u_end) pass(u0 + 4 * MT, kx, kc, mine + TILE, mine);
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // the newest key and value go into their slot (every reader took them from the new rows)
  if (kn && hc == 0 && vis.count > 0 && u_beg < vis.count && u_end == vis.count) {
    const int64_t at_slot = slot(vis.count - 1);
    for (int e = threadIdx.x; e < p.d / 4; e += 256) {   // 8 bytes a thread: keys, then values
      const bool isv = e >= p.d / 8;
      const int x = 8 * (isv ? e - p.d / 8 : e);
      *(uint4*)((isv ? V + at_slot * p.vp : K + at_slot * p.kp) + x) = *(const uint4*)((isv ? vn : kn) + x);
    }
  }
  // the block's waves joined through LDS
  __syncthreads();
  float* so = (float*)lds;   // [4][HEADS][LDO]
  if (c < nh) {
#pragma unroll
    for (int x = 0; x < NV; ++x) *(float4*)&so[(wave * HEADS + c) * LDO + 16 * x + 4 * g] = make_float4(o[x][0], o[x][1], o[x][2], o[x][3]);
    if (g == 0) { s_m[wave][c] = m; s_l[wave][c] = l; }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nh * (D / 4); e += 256) {
    const int hh = e / (D / 4), x = 4 * (e - hh * (D / 4));
    if (x >= p.d) continue;
    const float mm = fmaxf(fmaxf(s_m[0][hh], s_m[1][hh]), fmaxf(s_m[2][hh], s_m[3][hh]));
    float ll = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = s_m[w][hh] == -INFINITY ? (s_l[w][hh] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f((s_m[w][hh] - mm) * cs);
      const float4 v = *(const float4*)&so[(w * HEADS + hh) * LDO + x];
      ll += f * s_l[w][hh];
      a.x += f * v.x; a.y += f * v.y; a.z += f * v.z; a.w += f * v.w;
    }
    if (p.splits == 1) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      bf16_t* out = (bf16_t*)p.out + r * p.ldo + (int64_t)(h0 + hh) * p.d + x;
      out[0] = f32_to_bf16(a.x * inv); out[1] = f32_to_bf16(a.y * inv); out[2] = f32_to_bf16(a.z * inv); out[3] = f32_to_bf16(a.w * inv);
    } else {
      float* part = p.part + (((int64_t)r * p.H + h0 + hh) * p.splits + split) * (p.d + 2);
      part[x] = a.x; part[x + 1] = a.y; part[x + 2] = a.z; part[x + 3] = a.w;
      if (x == 0) { part[p.d] = mm * cs * (1.f / LOG2E); part[p.d + 1] = ll; }
    }
  }
}

// one block per (sequence, head): a thread adds one column over every second split
template <typename T>
__global__ __launch_bounds__(256) void step_join_kernel(StepParams p) {
  __shared__ float f[MAX_SPLITS], red[MAXD + 1];
  const int64_t rh = blockIdx.x;
  const int r = (int)(rh / p.H), h = (int)(rh - (int64_t)r * p.H), lane = threadIdx.x & 63;
  const float* part = p.part + rh * p.splits * (p.d + 2);
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, part[(int64_t)s * (p.d + 2) + p.d]);
  m = wave_max(m);
  for (int s = threadIdx.x; s < p.splits; s += 256) {
    const float ms = part[(int64_t)s * (p.d + 2) + p.d];
    f[s] = ms == -INFINITY ? 0.f : expf(ms - m);
  }
  __syncthreads();
  for (int s = lane; s < p.splits; s += 64) l += f[s] * part[(int64_t)s * (p.d + 2) + p.d + 1];
  l = wave_sum(l);
  const int col = threadIdx.x & (MAXD - 1), half = threadIdx.x / MAXD;
  float a = 0.f;
  if (col < p.d)
    for (int s = half; s < p.splits; s += 2) a += f[s] * part[(int64_t)s * (p.d + 2) + col];
  if (half) red[col] = a;
  __syncthreads();
  if (!half && col < p.d)
    ((T*)p.out)[r * p.ldo + (int64_t)h * p.d + col] = Cvt<T>::from_f32(l == 0.f ? 0.f : (a + red[col]) / l);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Splits: enough blocks to give every CU two, each with at least one pass of its four waves.
void plan(StepParams& p, bool mfma) {
  const int64_t most = std::min<int64_t>((int64_t)p.window + p.sinks, p.cap), pass = 4 * (mfma ? MT : KT);
  const int64_t blocks = (int64_t)p.R * (mfma ? p.G * ((p.H / p.G + HEADS - 1) / HEADS) : p.H);
  const int64_t want = std::min<int64_t>(MAX_SPLITS, 2 * sk_num_cus() / std::max<int64_t>(1, blocks));
  const int64_t passes = (most + pass - 1) / pass, splits = std::max<int64_t>(1, std::min(want, passes));
  p.per = (int)((passes + splits - 1) / splits * pass);
  p.splits = (int)((most + p.per - 1) / p.per);
}

int64_t ws_floats(const StepParams& p) { return p.splits > 1 ? (int64_t)p.R * p.H * p.splits * (p.d + 2) : 0; }

}  // namespace

extern "C" int64_t skhip_window_attn_step_ws_floats(int R, int n_head, int n_kv, int d, int cap, int window, int sinks) {
  if (R <= 0 || n_head <= 0 || n_kv <= 0 || d <= 0 || cap <= 0 || window < 1 || sinks < 0) return 0;
  StepParams p = {};
  p.R = R; p.H = n_head; p.G = n_kv; p.d = d; p.cap = cap; p.window = window; p.sinks = sinks;
  if (n_head % n_kv) return 0;
  // the larger of the two paths' needs: which one a call takes depends on its pointers and strides
  plan(p, false);
  const int64_t plain = ws_floats(p);
  plan(p, true);
  return std::max(plain, ws_floats(p));
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
  const bool mfma = dtype == SK_BF16 && rows16 && scale != 0.f && scale - scale == 0.f;
  plan(p, mfma);
  if (ws_floats(p) > 0 && (!workspace || workspace_floats < ws_floats(p))) {
    sk_set_error("%s: workspace of %lld floats needed", who, (long long)ws_floats(p));
    return SK_ERR_WORKSPACE;
  }
  const int chunks = (n_head / n_kv + HEADS - 1) / HEADS;
  const dim3 grid(p.splits, mfma ? n_kv * chunks : n_head, R);
  if (mfma && d <= 64) hipLaunchKernelGGL((step_mfma_kernel<64>), grid, dim3(256), 0, stream, p, chunks);
  else if (mfma) hipLaunchKernelGGL((step_mfma_kernel<128>), grid, dim3(256), 0, stream, p, chunks);
  else if (dtype == SK_BF16) hipLaunchKernelGGL((step_kernel<bf16_t>), grid, dim3(256), 0, stream, p, (int)rows16);
  else hipLaunchKernelGGL((step_kernel<float>), grid, dim3(256), 0, stream, p, (int)rows16);
  if (p.splits > 1) {
    const dim3 join((unsigned)(R * n_head));
    if (dtype == SK_BF16) hipLaunchKernelGGL((step_join_kernel<bf16_t>), join, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((step_join_kernel<float>), join, dim3(256), 0, stream, p);
  }
  SK_CHECK_LAUNCH(who);
  return SK_OK;
}
