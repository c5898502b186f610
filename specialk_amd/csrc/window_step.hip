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
#include "window_attn.h"
#include <algorithm>

namespace {

constexpr int MAXD = 128;
constexpr int KT = 64;   // keys per pass of a wave: one per lane

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

// one wave per (sequence, head)
template <typename T>
__global__ __launch_bounds__(256) void step_join_kernel(StepParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t rh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (rh >= (int64_t)p.R * p.H) return;
  const int r = (int)(rh / p.H), h = (int)(rh - (int64_t)r * p.H);
  const float* part = p.part + rh * p.splits * (p.d + 2);
  float m = -INFINITY;
  for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, part[(int64_t)s * (p.d + 2) + p.d]);
  m = wave_max(m);
  float l = 0.f, a0 = 0.f, a1 = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float* x = part + (int64_t)s * (p.d + 2);
    const float f = x[p.d] == -INFINITY ? 0.f : expf(x[p.d] - m);
    l += f * x[p.d + 1];
    if (lane < p.d) a0 += f * x[lane];
    if (lane + 64 < p.d) a1 += f * x[lane + 64];
  }
  T* out = (T*)p.out + r * p.ldo + (int64_t)h * p.d;
  if (lane < p.d) out[lane] = Cvt<T>::from_f32(l == 0.f ? 0.f : a0 / l);
  if (lane + 64 < p.d) out[lane + 64] = Cvt<T>::from_f32(l == 0.f ? 0.f : a1 / l);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Splits: enough blocks for two rounds of the chip, each with at least one pass of its four waves.
void plan(StepParams& p) {
  const int64_t most = std::min<int64_t>((int64_t)p.window + p.sinks, p.cap), pass = 4 * KT;
  const int64_t blocks = (int64_t)p.R * p.H, want = std::max<int64_t>(1, 2 * sk_num_cus() / std::max<int64_t>(1, blocks));
  const int64_t passes = (most + pass - 1) / pass, splits = std::max<int64_t>(1, std::min(want, passes));
  p.per = (int)((passes + splits - 1) / splits * pass);
  p.splits = (int)((most + p.per - 1) / p.per);
}

}  // namespace

extern "C" int64_t skhip_window_attn_step_ws_floats(int R, int n_head, int n_kv, int d, int cap, int window, int sinks) {
  if (R <= 0 || n_head <= 0 || n_kv <= 0 || d <= 0 || cap <= 0 || window < 1 || sinks < 0) return 0;
  StepParams p = {};
  p.R = R; p.H = n_head; p.G = n_kv; p.d = d; p.cap = cap; p.window = window; p.sinks = sinks;
  plan(p);
  return p.splits > 1 ? (int64_t)R * n_head * p.splits * (d + 2) : 0;
}

extern "C" int skhip_window_attn_step(const void* q, const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                                      void* out, const int32_t* kv_len, int R, int n_head, int n_kv, int d, int cap,
                                      int64_t ldq, int64_t ld_new, int64_t ldo, int64_t k_row, int64_t k_pos, int64_t v_row,
                                      int64_t v_pos, float scale, int window, int sinks, float* workspace,
                                      int64_t workspace_floats, int dtype, void* stream_) {
  const char* who = "skhip_window_attn_step";
  hipStream_t stream = (hipStream_t)stream_;
  SK_CHECK_ARG(dtype == SK_F32 || dtype == SK_BF16, "%s: bad dtype %d", who, dtype);
  SK_CHECK_ARG(R >= 0 && R <= 65535 && n_head > 0 && n_head <= 65535 && n_kv > 0, "%s: bad shape", who);
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
  plan(p);
  if (p.splits > 1 && (!workspace || workspace_floats < (int64_t)R * n_head * p.splits * (d + 2))) {
    sk_set_error("%s: workspace of %lld floats needed", who, (long long)R * n_head * p.splits * (d + 2));
    return SK_ERR_WORKSPACE;
  }
  const int per = dtype == SK_BF16 ? 8 : 4;
  const int vec = d % per == 0 && (k_row | k_pos) % per == 0 && aligned16(k_cache) && (!k_new || (aligned16(k_new) && ld_new % per == 0));
  dim3 grid(p.splits, n_head, R);
  const unsigned join = (unsigned)(((int64_t)R * n_head + 3) / 4);
  if (dtype == SK_BF16) {
    hipLaunchKernelGGL((step_kernel<bf16_t>), grid, dim3(256), 0, stream, p, vec);
    if (p.splits > 1) hipLaunchKernelGGL((step_join_kernel<bf16_t>), dim3(join), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((step_kernel<float>), grid, dim3(256), 0, stream, p, vec);
    if (p.splits > 1) hipLaunchKernelGGL((step_join_kernel<float>), dim3(join), dim3(256), 0, stream, p);
  }
  SK_CHECK_LAUNCH(who);
  return SK_OK;
}
