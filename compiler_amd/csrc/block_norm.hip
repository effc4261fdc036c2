// The norms around a block on gfx950, one pass over the residual stream:
//   u = h * rsqrt(mean(h^2) + eps) * w_post     (norm after the block; optional)
//   y = alpha * x + act(g) * u                  (gate optional: none, sigmoid, tanh)
//   n = y * rsqrt(mean(y^2) + eps) * w_pre      (norm before the next; optional)
// per row, in fp32 throughout: n comes from y before y's rounding, and each
// output rounds once.  1 / sqrt as in the row norms.
namespace g950 {

// sigmoid(g) = 1 / (1 + e^-g); tanh(g) = (1 - e^-2|g|) / (1 + e^-2|g|) with g's
// sign, near 0 (where the difference cancels) the odd series to g^7 (next term
// 62 / 2835 g^9: below 2e-8 of g for |g| < 0.18)
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

}  // namespace g950

extern "C" __global__ __launch_bounds__(256) void g950_block_norm_general(const g950::BlockNormArgs a) {
  g950::block_norm_general_body(a);
}
