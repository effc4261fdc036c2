// Attention over a paged cache of 4-bit rows (kv_append.hip's format) on
// gfx950.  Query i of sequence b (rows cu[b] ..) sees keys j of that sequence's
// used[b] with i + used - n - left <= j <= i + used - n + right (n its queries;
// an unbounded side has no limit) whose page the pool holds:
//   S = scale q.K, O = softmax(S) V, LSE = log(sum(exp(S)));
// a row that sees no key gets O = 0 and LSE = +inf.
namespace g950 {

struct Int4Seq {
  int q0, nq, nk;  // first query row, queries, keys
};

// Sequence z's rows and keys; rows outside q or keys outside the table count
// as none.
__device__ __forceinline__ Int4Seq int4_seq(const AttnInt4Args& p, int z) {
  Int4Seq s;
  const int b0 = p.cu[z], b1 = p.cu[z + 1];
  s.q0 = b0;
  s.nq = b0 >= 0 && b1 >= b0 && b1 <= p.T ? b1 - b0 : 0;
  const long long held = (long long)p.max_pages * p.block_size;
  const int used = p.used[z];
  s.nk = used < 0 ? 0 : (long long)used > held ? (int)held : used;
  return s;
}

// One wave per (query row, head): any D, page size, stride and alignment.
// Lanes take keys for the scores, dims for O.
__device__ __forceinline__ void attn_int4_general_body(const AttnInt4Args& p) {
  __shared__ float qs[256];
  __shared__ float pr[64], vo[64];
  __shared__ const uint8_t* vrow[64];
  const int lane = threadIdx.x;
  const int h = blockIdx.x % p.Hq, t = blockIdx.x / p.Hq;
  int b0 = 0, b1 = 0;
  const int z = kv_sequence(p.cu, p.B, p.T, t, b0, b1);
  if (z < 0 || t - b0 >= p.seqlen_q) return;
  const Int4Seq sq = int4_seq(p, z);
  const int hk = h / p.group;
  float qsum = 0.0f;
  for (int d = lane; d < p.D; d += 64) {
    const float x = load_as_f32(p.q, t * p.q_st + h * p.q_sh + d, p.dtype);
    qs[d] = x;
    qsum += x;
  }
  qsum = wave_reduce<OpSum>(qsum);
  __syncthreads();
  // window in 64 bits: lengths and limits may be any int
  const long long base = (long long)(t - b0) + p.used[z] - (b1 - b0);
  long long beg = p.left < 0 ? 0 : base - p.left, end = p.right < 0 ? sq.nk : base + p.right + 1;
  beg = beg < 0 ? 0 : beg;
  end = end > sq.nk ? sq.nk : end;
  float m = -__builtin_huge_valf(), l = 0.0f;
  float acc[4] = {};
  for (long long j0 = beg; j0 < end; j0 += 64) {
    const int j = (int)j0 + lane;
    float s = -__builtin_huge_valf();
    float sv = 0.0f, ov = 0.0f;
    const uint8_t* vr = nullptr;
    bool live = j0 + lane < end;
    if (live) {
      const int ph = p.table[(long long)z * p.table_s + j / p.block_size];
      live = ph >= 0 && ph < p.pages;
      if (live) {
        const int r = j % p.block_size;
        const uint8_t* kr = p.k + ph * p.k_p + r * p.k_r + hk * p.k_h;
        vr = p.v + ph * p.v_p + r * p.v_r + hk * p.v_h;
        const long long so = ph * p.ks_p + r * p.ks_r + hk * p.ks_h, wo = ph * p.vs_p + r * p.vs_r + hk * p.vs_h;
        float dot = 0.0f;
        for (int i = 0; i < p.D / 2; ++i) {
          const int c = kr[i];
          dot = fmaf(qs[2 * i], (float)((c & 15) - 8), dot);
          dot = fmaf(qs[2 * i + 1], (float)((c >> 4) - 8), dot);
        }
        s = fmaf(load_as_f32(p.ks, so, p.dtype), dot, load_as_f32(p.ks, so + 1, p.dtype) * qsum) * p.scale_log2;
        sv = load_as_f32(p.vs, wo, p.dtype);
        ov = load_as_f32(p.vs, wo + 1, p.dtype);
      }
    }
    const float mt = fmaxf(m, wave_reduce<OpMax>(s));
    const float mb = mt == -__builtin_huge_valf() ? 0.0f : mt;
    const float alpha = m == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(m - mb);
    const float e = live ? __builtin_amdgcn_exp2f(s - mb) : 0.0f;
    l = fmaf(l, alpha, wave_reduce<OpSum>(e));
    m = mt;
    __syncthreads();
    pr[lane] = live ? e * sv : 0.0f;
    vo[lane] = live ? e * ov : 0.0f;
    vrow[lane] = vr;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d >= p.D) break;
      float o = acc[i] * alpha;
      for (int n = 0; n < 64; ++n) {
        const uint8_t* r = vrow[n];
        if (!r) continue;
        const int c = (r[d >> 1] >> (4 * (d & 1))) & 15;
        o += fmaf(pr[n], (float)(c - 8), vo[n]);
      }
      acc[i] = o;
    }
  }
  const bool empty = !(l > 0.0f);  // zero or NaN
  const float inv = empty ? 1.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < p.D) store_from_f32(p.o, t * p.o_st + h * p.o_sh + d, p.dtype, acc[i] * inv);
  }
  if (lane == 0)
    p.lse[h * p.lse_h + t * p.lse_t] =
        empty ? __builtin_huge_valf() : (m + __log2f(l)) * 0.69314718055994530942f;
}

}  // namespace g950

extern "C" __global__ __launch_bounds__(64) void g950_attn_int4_general(const g950::AttnInt4Args p) {
  g950::attn_int4_general_body(p);
}
