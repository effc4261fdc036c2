// Attention of the nodes of drafted token trees over a paged cache on gfx950.
// Node i of sequence z (row cu[z] + i, n of them) has a parent among the nodes
// before it, or none (any other value); base = used[z] - n keys lie before the tree and the
// nodes' own behind them, node i's in cache row base + i, at position base + depth(i).
// It sees
//   the keys j < base, with a window those at positions j >= base + depth - left,
//   its own and the nodes above it, with a window up to `left` levels,
// whose page the pool holds: S = scale q.K, O = softmax(S) V, LSE = log(sum(exp(S))); a
// node that sees no key gets O = 0 and LSE = +inf.
namespace g950 {

struct TreeSeq {
  int q0, n, nq;  // first row, nodes, those of them that take part
  int base;       // keys before the tree; -n: none of the sequence's keys exist
};
__device__ __forceinline__ TreeSeq tree_seq(const int* cu, const int* used, int T, int most, int z) {
  TreeSeq s;
  const int b0 = cu[z], b1 = cu[z + 1];
  s.q0 = b0;
  s.n = b0 >= 0 && b1 >= b0 && b1 <= T ? b1 - b0 : 0;
  s.nq = min(s.n, most);
  s.base = max(used[z], 0) - s.n;
  return s;
}
// a node's parent, -1 if it has none
__device__ __forceinline__ int tree_parent(const int* parent, const TreeSeq& s, int i) {
  const int p = parent[s.q0 + i];
  return p >= 0 && p < i ? p : -1;
}

// The sequence that row t is a node of, -1: none.  (By each sequence's own bounds, which
// need not rise from one to the next.)
__device__ __forceinline__ int tree_sequence(const int* cu, int B, int T, int t) {
  const int lane = threadIdx.x & 63;
  for (int z0 = 0; z0 < B; z0 += 64) {
    const int z = min(z0 + lane, B - 1), b0 = cu[z], b1 = cu[z + 1];
    const uint64_t in = __ballot(b0 >= 0 && b0 <= t && t < b1 && b1 <= T);
    if (in) return min(z0 + __ffsll((unsigned long long)in) - 1, B - 1);
  }
  return -1;
}

// One wave per (node, head): any D, type, page size, stride and alignment.  Lanes take
// keys for the scores, dims for O; keys are taken from the last to the first, so that the
// way from the node to its root meets them in order.
__device__ __forceinline__ void attn_tree_general_body(const AttnTreeArgs& p) {
  __shared__ float qs[256];
  __shared__ float pr[64];
  __shared__ long long vrow[64];
  const int lane = threadIdx.x;
  const int h = blockIdx.x % p.Hq, t = blockIdx.x / p.Hq;
  const int z = tree_sequence(p.cu, p.B, p.T, t);
  if (z < 0) return;
  const TreeSeq sq = tree_seq(p.cu, p.used, p.T, p.seqlen_q, z);
  const int hk = h / p.group, i = t - sq.q0;
  if (i >= sq.nq) return;
  for (int d = lane; d < p.D; d += 64) qs[d] = load_as_f32(p.q, t * p.q_st + h * p.q_sh + d, p.dtype);
  __syncthreads();
  int lo = 0;
  if (p.left >= 0) {
    int depth = 0;
    for (int c = tree_parent(p.parent, sq, i); c >= 0; c = tree_parent(p.parent, sq, c)) ++depth;
    lo = max(0ll, (long long)sq.base + depth - p.left);
  }
  int cur = i, up = 0;  // next node of the way, levels above node i
  float m = -__builtin_huge_valf(), l = 0.0f;
  float acc[4] = {};
  const long long last = (long long)sq.base + i;  // its own key: none behind it is seen
  for (int j0 = last < 0 ? -1 : (int)(last / 64 * 64); j0 >= 0 && (j0 + 63 >= lo || cur >= 0); j0 -= 64) {
    // nodes of the way in this run of keys
    uint64_t way = 0;
    while (cur >= 0 && (long long)sq.base + cur >= j0) {
      if (p.left < 0 || up <= p.left) way |= 1ull << (sq.base + cur - j0);
      cur = tree_parent(p.parent, sq, cur);
      ++up;
    }
    const int j = j0 + lane;
    float s = -__builtin_huge_valf();
    long long vr = -1;
    if ((way >> lane & 1) || (j >= lo && j < sq.base)) {
      const int e = j / p.block_size;
      const int ph = e < p.max_pages ? p.table[(long long)z * p.table_s + e] : -1;
      if (ph >= 0 && ph < p.pages) {
        const int r = j % p.block_size;
        const long long kr = ph * p.k_p + r * p.k_r + hk * p.k_h;
        vr = ph * p.v_p + r * p.v_r + hk * p.v_h;
        float dot = 0.0f;
        for (int d = 0; d < p.D; ++d) dot = fmaf(qs[d], load_as_f32(p.k, kr + d, p.dtype), dot);
        s = dot * p.scale_log2;
      }
    }
    const bool live = vr >= 0;
    if (!__any(live)) continue;
    const float mt = fmaxf(m, wave_reduce<OpMax>(s));
    const float mb = mt == -__builtin_huge_valf() ? 0.0f : mt;
    const float alpha = m == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(m - mb);
    const float e = live ? __builtin_amdgcn_exp2f(s - mb) : 0.0f;
    l = fmaf(l, alpha, wave_reduce<OpSum>(e));
    m = mt;
    __syncthreads();
    pr[lane] = e;
    vrow[lane] = vr;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + 64 * u;
      if (d >= p.D) break;
      float o = acc[u] * alpha;
      for (int n = 0; n < 64; ++n)
        if (vrow[n] >= 0) o = fmaf(pr[n], load_as_f32(p.v, vrow[n] + d, p.dtype), o);
      acc[u] = o;
    }
  }
  const bool empty = !(l > 0.0f);  // zero or NaN
  const float inv = empty ? 1.0f : 1.0f / l;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int d = lane + 64 * u;
    if (d < p.D) store_from_f32(p.o, t * p.o_st + h * p.o_sh + d, p.dtype, acc[u] * inv);
  }
  if (lane == 0)
    p.lse[h * p.lse_h + t * p.lse_t] =
        empty ? __builtin_huge_valf() : (m + __log2f(l)) * 0.69314718055994530942f;
}

}  // namespace g950

extern "C" __global__ __launch_bounds__(64) void g950_attn_tree_general(const g950::AttnTreeArgs p) {
  g950::attn_tree_general_body(p);
}
