// Verification of drafted token trees against the target's probabilities on
// gfx950.  Row cu[z] + i of the target's p holds its distribution after node i
// of sequence z, the same row of the draft's q the one that node i's children
// were drawn from.  From the root (node 0), the children of the node reached
// are tested in order with their own random number u; the first one accepted is
// the next node of the path.  What is left of p after k refusals, not
// normalised, is
//   R_k = max(R_{k-1} - (S_{k-1} / Q_{k-1}) q, 0) = max(p - A_k q, 0),  A_k = sum_{j<k} S_j / Q_j:
// clamped differences by multiples of one q >= 0 compose, so one number stands
// for all refusals, and what a refused token keeps is 0 by itself.
//   accept x if u q(x) S < max(p(x) - A q(x), 0) Q,    at first A = 0, S = Q = 1
//   else  A += S / Q,  S = sum max(p - A q, 0),  Q = max(Q - q(x), 2^-24) if siblings
//   were drawn without replacement.
// (q(x) / Q is then what the draft had left when it drew x; 2^-24 stands for a draft
// used up to rounding.)  Without q a child was chosen, not drawn: q is 1 at its token, so
// a refusal takes the token out, S -= p(x).  The next token is the first v with
// sum_{w <= v} R(w) > r sum R; where nothing is left (S = 0), p's row itself is taken.  All sums are held in
// 64 bits: a comparison falls otherwise than the formula's only where both sides agree
// to 2^-45 or so.
namespace g950 {

constexpr int VERIFY_THREADS = 1024, VERIFY_WAVES = VERIFY_THREADS / 64;

// a probability: below zero and NaN count as none
template <typename T>
__device__ __forceinline__ double verify_value(T x) {
  if constexpr (std::is_same_v<T, float>) return fmax((double)x, 0.0);
  else if constexpr (std::is_same_v<T, bf16_t>) return fmax((double)bf16_to_f32(x.bits), 0.0);
  else return fmax((double)f16_to_f32(x.bits), 0.0);
}

__device__ __forceinline__ double verify_shfl_up(double v, int by) { return __shfl_up(v, by); }

// One workgroup per sequence.
template <typename T>
__device__ __forceinline__ void verify_tree_body(const VerifyArgs& a) {
  __shared__ double px[TREE_NODES], qx[TREE_NODES];
  __shared__ float us[TREE_NODES];
  __shared__ int tok[TREE_NODES], gone[TREE_NODES];
  __shared__ short par[TREE_NODES];
  __shared__ double seg[VERIFY_WAVES + 1];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int z = blockIdx.x;
  const int b0 = a.cu[z], b1 = a.cu[z + 1];
  const int n = b0 >= 0 && b1 >= b0 && b1 <= a.T ? min(b1 - b0, TREE_NODES) : 0;
  int* path = a.path + z * a.path_z;
  if (n == 0) {
    for (int i = tid; i < a.L; i += VERIFY_THREADS) path[i] = -1;
    if (tid == 0) {
      a.count[z * a.count_z] = 0;
      if (a.token64) ((long long*)a.next)[z * a.next_z] = -1;
      else ((int*)a.next)[z * a.next_z] = -1;
    }
    return;
  }
  const T* P = (const T*)a.target;
  const T* Q = (const T*)a.draft;
  // every node's token, its probability after its parent and there in the draft
  for (int i = tid; i < n; i += VERIFY_THREADS) {
    int p = a.parent[b0 + i];
    p = i > 0 && p >= 0 && p < i ? p : -1;
    const long long x = a.token64 ? ((const long long*)a.tokens)[b0 + i] : ((const int*)a.tokens)[b0 + i];
    const bool in = p >= 0 && x >= 0 && x < a.V;
    par[i] = (short)p;
    tok[i] = in ? (int)x : -1;
    us[i] = a.u[b0 + i];
    px[i] = in ? verify_value(P[(b0 + p) * a.t_row + x]) : 0.0;
    qx[i] = !Q ? 1.0 : in ? verify_value(Q[(b0 + p) * a.d_row + x]) : 0.0;
  }
  __syncthreads();
  int cur = 0, count = 1, refused = 0;
  double A = 0.0, S = 1.0, rest = 1.0;
  // what is left of column v
  auto left = [&](const T* pr, const T* qr, int v) {
    double r = verify_value(pr[v]);
    if (qr) return fmax(r - A * verify_value(qr[v]), 0.0);
    for (int k = 0; k < refused; ++k) r = gone[k] == v ? 0.0 : r;
    return r;
  };
  const int per = (a.V + VERIFY_WAVES - 1) / VERIFY_WAVES;  // columns of a wave
  // seg[w]: what is left in the columns of the waves before w
  auto sum = [&]() {
    const T* pr = P + (long long)(b0 + cur) * a.t_row;
    const T* qr = Q && A > 0.0 ? Q + (long long)(b0 + cur) * a.d_row : nullptr;
    const long long end = min((long long)(wave + 1) * per, (long long)a.V);
    double s = 0.0;
    for (long long v = (long long)wave * per + lane; v < end; v += 64) s += left(pr, qr, (int)v);
    for (int k = 32; k; k >>= 1) s += __shfl_xor(s, k);
    __syncthreads();
    if (lane == 0) seg[wave + 1] = s;
    __syncthreads();
    if (tid == 0) {
      seg[0] = 0.0;
      for (int w = 0; w < VERIFY_WAVES; ++w) seg[w + 1] += seg[w];
    }
    __syncthreads();
    return seg[VERIFY_WAVES];
  };
  bool known = false;  // seg holds the sums of this node with this A
  for (int i = 1; i < n && count < a.L; ++i) {
    if (par[i] != cur) continue;
    double r = Q ? fmax(px[i] - A * qx[i], 0.0) : px[i];
    if (!Q)
      for (int k = 0; k < refused; ++k) r = gone[k] == tok[i] ? 0.0 : r;
    if ((double)us[i] * qx[i] * S < r * rest) {
      if (tid == 0) path[count] = i;
      ++count;
      cur = i;
      refused = 0;
      A = 0.0;
      S = rest = 1.0;
      known = false;
    } else if (Q) {
      A += S / rest;
      S = sum();
      known = true;
      if (a.distinct) rest = fmax(rest - qx[i], 0x1p-24);
    } else {
      S -= r;
      __syncthreads();
      if (tid == 0) gone[refused] = tok[i];
      ++refused;
      __syncthreads();
    }
  }
  double total = known ? S : sum();
  if (!(total > 0.0)) {
    A = 0.0;
    refused = 0;
    total = sum();
  }
  // the first column whose sum passes the random number's share
  const double want = (double)a.last[z] * total;
  int w = 0;
  while (w + 1 < VERIFY_WAVES && !(seg[w + 1] > want)) ++w;
  while (w > 0 && !(seg[w + 1] > seg[w])) --w;  // (a share past the end)
  const T* pr = P + (long long)(b0 + cur) * a.t_row;
  const T* qr = Q && A > 0.0 ? Q + (long long)(b0 + cur) * a.d_row : nullptr;
  if (tid == 0) found = -1;
  __syncthreads();
  if (wave == 0) {
    double before = seg[w];
    const long long end = min((long long)(w + 1) * per, (long long)a.V);
    int some = -1, hit = -1;  // last column with something left; the one wanted
    for (long long v0 = (long long)w * per; v0 < end && hit < 0; v0 += 64) {
      const long long v = v0 + lane;
      const double r = v < end ? left(pr, qr, (int)v) : 0.0;
      double s = r;
      for (int k = 1; k < 64; k <<= 1) {
        const double t = __shfl_up(s, k);
        s += lane >= k ? t : 0.0;
      }
      const uint64_t over = __ballot(r > 0.0 && before + s > want), any = __ballot(r > 0.0);
      if (over) hit = (int)v0 + __ffsll((unsigned long long)over) - 1;
      if (any) some = (int)v0 + 63 - __clzll((long long)any);
      before += __shfl(s, 63);
    }
    if (lane == 0) found = hit >= 0 ? hit : some >= 0 ? some : 0;
  }
  __syncthreads();
  for (int i = count + tid; i < a.L; i += VERIFY_THREADS) path[i] = -1;
  if (tid == 0) {
    path[0] = 0;
    a.count[z * a.count_z] = count;
    if (a.token64) ((long long*)a.next)[z * a.next_z] = found;
    else ((int*)a.next)[z * a.next_z] = found;
  }
}

}  // namespace g950

#define G950_VERIFY(TNAME, T)                                                                                 \
  extern "C" __global__ __launch_bounds__(1024) void g950_verify_tree_##TNAME(const g950::VerifyArgs a) {    \
    g950::verify_tree_body<T>(a);                                                                             \
  }
G950_VERIFY(f32, float)
G950_VERIFY(bf16, g950::bf16_t)
G950_VERIFY(f16, g950::f16_t)
