// The norms around a block on gfx950, one pass over the residual stream:
//   u = h * rsqrt(mean(h^2) + eps) * w_post     (norm after the block; optional)
//   y = alpha * x + act(g) * u                  (gate optional: none, sigmoid, tanh)
//   n = y * rsqrt(mean(y^2) + eps) * w_pre      (norm before the next; optional)
// per row, in fp32 throughout: n comes from y before y's rounding, and each
// output rounds once.  1 / sqrt as in the row norms.
namespace g950 {

// sigmoid(g) = 1 / (1 + e^-g); tanh(g) = (1 - e^-2|g|) / (1 + e^-2|g|) with g's
// sign, near 0 (where the difference cancels) the odd series to g^7 (next term
// 62 / 2835 g^9: below 2.5e-8 of g for |g| < 0.18)
__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == 0) return g;
  if (act == 1) return 1.0f / (1.0f + __expf(-g));
  const float a = fabsf(g), e = __expf(-2.0f * a), g2 = g * g;
  const float big = copysignf((1.0f - e) / (1.0f + e), g);
  const float small = g * fmaf(g2, fmaf(g2, fmaf(g2, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  return a < 0.18f ? small : big;
}

// One workgroup per row, the row read once per sum: any length and alignment.
// y may be x and n may be h: an element is read last by the thread that
// writes it.
__device__ __forceinline__ void block_norm_general_body(const BlockNormArgs& a) {
  __shared__ float scratch[4];
  const long long r = blockIdx.x;
  const int dt = a.dtype;
  float rh = 1.0f;
  if (a.w_post) {
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      const float v = load_as_f32(a.h, r * a.h_row + c, dt);
      s = fmaf(v, v, s);
    }
    rh = 1.0f / sqrtf(block_reduce<OpSum, 256>(s, scratch) / (float)a.cols + a.eps);
  }
  auto value = [&](int c) {
    float u = load_as_f32(a.h, r * a.h_row + c, dt);
    if (a.w_post) u = u * rh * load_as_f32(a.w_post, c, dt);
    if (a.gate) u *= gate_act(load_as_f32(a.gate, r * a.g_row + c * a.g_col, dt), a.act);
    return fmaf(a.alpha, load_as_f32(a.x, r * a.x_row + c, dt), u);
  };
  float ry = 0.0f;
  if (a.w_pre) {
    float s = 0.0f;
    for (int c = threadIdx.x; c < a.cols; c += 256) {
      const float v = value(c);
      s = fmaf(v, v, s);
    }
    ry = 1.0f / sqrtf(block_reduce<OpSum, 256>(s, scratch) / (float)a.cols + a.eps);
  }
  for (int c = threadIdx.x; c < a.cols; c += 256) {
    const float v = value(c);
    store_from_f32(a.y, r * a.y_row + c, dt, v);
    if (a.w_pre) store_from_f32(a.n, r * a.n_row + c, dt, v * ry * load_as_f32(a.w_pre, c, dt));
  }
}

// ---- one workgroup per row, the row in registers: x and h are read once, y and n
// written once, so a large batch is bound by HBM: bfloat16 [8191, 3000] with a gate per
// channel, 197 MB in 36.9 us, 5.3 TB/s; fp32 [4096, 4096] with a gate for every value, 335 MB
// in 59.6 us, 5.6 TB/s (a plain copy: 6.0; the general kernel, which reads the row three
// times over: 233 and 155 us).  16 rows of 4096 take 4.2 us: launch, load, two sums across
// the workgroup.
// 16 bytes of a row at any element alignment (the hardware takes unaligned
// 16-byte accesses: rows of odd length and all alignments share one kernel)
typedef uint32_t u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
struct BnVec {
  static constexpr int V = 16 / sizeof(T);
  using raw_any = std::conditional_t<sizeof(T) == 4, u32x4_any4, u32x4_any2>;
  static __device__ __forceinline__ float to(uint32_t bits) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
    else if constexpr (std::is_same_v<T, bf16_t>) return bf16_to_f32((uint16_t)bits);
    else return f16_to_f32((uint16_t)bits);
  }
  static __device__ __forceinline__ uint32_t from(float v) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(v);
    else if constexpr (std::is_same_v<T, bf16_t>) return f32_to_bf16(v);
    else return f32_to_f16(v);
  }
  using word = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
  // vector j of a row of `cols` elements; the last may be a part (zero filled)
  static __device__ __forceinline__ u32x4 load(const void* row, int j, int cols, bool once) {
    const word* p = (const word*)row + j * V;
    if ((j + 1) * V <= cols) {
      const raw_any* q = (const raw_any*)p;
      const raw_any r = once ? __builtin_nontemporal_load(q) : *q;
      return (u32x4){r[0], r[1], r[2], r[3]};
    }
    u32x4 r = {};
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (j * V + e < cols) r[e * (int)sizeof(T) / 4] |= (uint32_t)p[e] << (8 * (e * (int)sizeof(T) % 4));
    return r;
  }
  static __device__ __forceinline__ float get(const u32x4& r, int e) {
    if constexpr (sizeof(T) == 4) return to(r[e]);
    else return to((r[e / 2] >> (16 * (e & 1))) & 0xFFFFu);
  }
  static __device__ __forceinline__ void store(void* row, int j, int cols, const float* v) {
    word* p = (word*)row + j * V;
    if ((j + 1) * V <= cols) {
      raw_any r;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (sizeof(T) == 4) r[w] = from(v[w]);
        else r[w] = from(v[2 * w]) | from(v[2 * w + 1]) << 16;
      }
      *(raw_any*)p = r;
      return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (j * V + e < cols) p[e] = (word)from(v[e]);
  }
};

// GATE: 0 none, 1 a vector of gates beside h (per channel or full), 2 one per row
template <typename T, int ITEMS, int BLOCK, int GATE>
__device__ __forceinline__ void block_norm_body(const BlockNormArgs& a) {
  using M = BnVec<T>;
  constexpr int V = M::V;
  __shared__ float scratch[BLOCK / 64 > 0 ? BLOCK / 64 : 1];
  const int tid = threadIdx.x, cols = a.cols;
  const int nv = (cols + V - 1) / V;
  // the weights and gates come in while the row does; long rows have no
  // registers for them until the row is summed
  constexpr bool EARLY = ITEMS <= 2;
  const long long r = blockIdx.x;
  const char* xr = (const char*)a.x + r * a.x_row * (long long)sizeof(T);
  const char* hr = (const char*)a.h + r * a.h_row * (long long)sizeof(T);
  const char* gr = (const char*)a.gate + r * a.g_row * (long long)sizeof(T);
  char* yr = (char*)a.y + r * a.y_row * (long long)sizeof(T);
  char* nr = (char*)a.n + r * a.n_row * (long long)sizeof(T);
  u32x4 x[ITEMS], h[ITEMS], g[GATE == 1 ? ITEMS : 1], wo[ITEMS], wi[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int j = tid + i * BLOCK;
    x[i] = h[i] = wo[i] = wi[i] = g[GATE == 1 ? i : 0] = (u32x4){};
    if (j < nv) {
      h[i] = M::load(hr, j, cols, true);
      x[i] = M::load(xr, j, cols, true);
      if constexpr (GATE == 1 && EARLY) g[i] = M::load(gr, j, cols, false);
    }
  }
  auto weights = [&](const void* w, u32x4(&to)[ITEMS]) {
    if (w) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (tid + i * BLOCK < nv) to[i] = M::load(w, tid + i * BLOCK, cols, false);
    }
  };
  if constexpr (EARLY) {
    weights(a.w_post, wo);
    weights(a.w_pre, wi);
  }
  float one = 1.0f;
  if constexpr (GATE == 2) one = gate_act(load_as_f32(gr, 0, a.dtype), a.act);
  float rh = 1.0f;
  if (a.w_post) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = M::get(h[i], e);
        s = fmaf(v, v, s);
      }
    rh = 1.0f / sqrtf(block_reduce<OpSum, BLOCK>(s, scratch) / (float)cols + a.eps);
  }
  if constexpr (!EARLY) {
    weights(a.w_post, wo);
    if constexpr (GATE == 1) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (tid + i * BLOCK < nv) g[i] = M::load(gr, tid + i * BLOCK, cols, false);
    }
  }
  float y[ITEMS][V];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float u = M::get(h[i], e);
      if (a.w_post) u = u * rh * M::get(wo[i], e);
      if constexpr (GATE == 1) u *= gate_act(M::get(g[i], e), a.act);
      if constexpr (GATE == 2) u *= one;
      y[i][e] = fmaf(a.alpha, M::get(x[i], e), u);  // (past the row: 0)
      s = fmaf(y[i][e], y[i][e], s);
    }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i)
    if (tid + i * BLOCK < nv) M::store(yr, tid + i * BLOCK, cols, y[i]);
  if (!a.w_pre) return;
  if constexpr (!EARLY) weights(a.w_pre, wi);
  const float ry = 1.0f / sqrtf(block_reduce<OpSum, BLOCK>(s, scratch) / (float)cols + a.eps);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) y[i][e] = y[i][e] * ry * M::get(wi[i], e);
    if (tid + i * BLOCK < nv) M::store(nr, tid + i * BLOCK, cols, y[i]);
  }
}

}  // namespace g950

extern "C" __global__ __launch_bounds__(256) void g950_block_norm_general(const g950::BlockNormArgs a) {
  g950::block_norm_general_body(a);
}

#define G950_BN_GATE(TNAME, T, ITEMS, BLOCK, GATE)                                          \
  extern "C" __global__ __launch_bounds__(BLOCK) void                                       \
      g950_block_norm_##TNAME##_i##ITEMS##_b##BLOCK##_g##GATE(const g950::BlockNormArgs a) { \
    g950::block_norm_body<T, ITEMS, BLOCK, GATE>(a);                                        \
  }
#define G950_BN(TNAME, T, ITEMS, BLOCK)       \
  G950_BN_GATE(TNAME, T, ITEMS, BLOCK, 0)     \
  G950_BN_GATE(TNAME, T, ITEMS, BLOCK, 1)     \
  G950_BN_GATE(TNAME, T, ITEMS, BLOCK, 2)
#define G950_BN_SET(TNAME, T)  \
  G950_BN(TNAME, T, 1, 64)     \
  G950_BN(TNAME, T, 2, 64)     \
  G950_BN(TNAME, T, 1, 256)    \
  G950_BN(TNAME, T, 2, 256)    \
  G950_BN(TNAME, T, 2, 512)    \
  G950_BN(TNAME, T, 2, 1024)   \
  G950_BN(TNAME, T, 4, 1024)
G950_BN_SET(f32, float)
G950_BN_SET(bf16, g950::bf16_t)
G950_BN_SET(f16, g950::f16_t)
