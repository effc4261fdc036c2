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
//
// A test needs four numbers; a refusal needs its node's two rows, and the next test waits
// for their sum: a chain of passes over one pair of rows after the other (a megabyte each at
// 128000 tokens in fp32), which one CU streams at some 100 GB/s.  So a sequence's columns are cut into
// `parts`, one workgroup each, all of which follow the path on their own and tell each other
// their sums.  Bound by that chain: 2.8 us a refusal, 3.5 where 16 trees share the chip (waves'
// sums, barriers, a store and a load past the L2); one workgroup takes 11 over 32000 columns in
// fp32, 42 over 128000.  One tree of 26 nodes over 32000 columns 1.7 + 9.8 us (gather and parts), 16 of
// 9 to 26 over 128000, siblings distinct, 4.0 + 24.8; 32 chosen ones over 50257 in bfloat16 2.6 + 12.6, by time stamps in a
// workgroup, each tree's mean: nodes 0.7, walk 2.6 (the longest path's 5), rows 2.4, sums told and taken 1.6, the
// token 0.7; the last tree's is there 11 after the first workgroup's start.  Rows of which a wave's share is more
// than 1024 fp32 columns are read again for every sum: 32 trees over 128000 4.8 + 51, 16 over 151936 4.8 + 33.  60 refusals of one root in a row 171 us over 32000 columns as over 128000 (one workgroup
// 714 and 2620), 120 of them 335.
//   * A sum is told in one 64-bit word, by a relaxed atomic, in a place of its own for every
//     (sequence, round, part); the launch before empties the places (a pattern that no sum
//     has).  So nothing else needs to be ordered, and a place is never written twice with
//     different values.  A sequence of n nodes has n rounds at most: one
//     for each node refused (never the root, and none twice) and one more where the path ends (where
//     children are chosen: up to two there, and no others).
//   * A workgroup waits for a sum for a bounded time only, then adds up that part itself,
//     in the same order, to the same bits: no workgroup depends on another one's being on
//     the chip.
//   * The part in which the random number's share falls belongs to one workgroup, which
//     finds the token.
namespace g950 {

constexpr int VERIFY_THREADS = 256, VERIFY_WAVES = VERIFY_THREADS / 64;
constexpr int VERIFY_SPINS = 64;  // looks at what others tell, about a microsecond each
constexpr uint64_t VERIFY_EMPTY = ~0ull;

// 16 bytes of a row, which may begin at any element
typedef u32x4 __attribute__((aligned(4))) verify_word4;
typedef u32x4 __attribute__((aligned(2))) verify_word2;
// a probability: below zero and NaN count as none
__device__ __forceinline__ double verify_value(float x) { return (double)fmaxf(x, 0.0f); }
__device__ __forceinline__ double verify_value(bf16_t x) { return verify_value(bf16_to_f32(x.bits)); }
__device__ __forceinline__ double verify_value(f16_t x) { return verify_value(f16_to_f32(x.bits)); }
template <typename T>
__device__ __forceinline__ double verify_element(const u32x4& w, int e) {
  if constexpr (sizeof(T) == 4) return verify_value(__uint_as_float(w[e]));
  else return verify_value(T{(uint16_t)(w[e / 2] >> (16 * (e & 1)))});
}

// sums of `v` over the lanes up to the own one
template <int CTRL, int ROWS>
__device__ __forceinline__ double verify_dpp(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)w, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(w >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double verify_scan(double v) {
  v += verify_dpp<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += verify_dpp<0x112, 0xF>(v);
  v += verify_dpp<0x114, 0xF>(v);
  v += verify_dpp<0x118, 0xF>(v);
  v += verify_dpp<0x142, 0xA>(v);  // row_bcast 15, 31
  v += verify_dpp<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ double verify_lane(double v, int lane) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)w, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(w >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A node's token and its probabilities after its parent.
template <typename T>
__device__ __forceinline__ void verify_node(const VerifyArgs& a, int b0, int i, int& p, int& x, double& px, double& qx) {
  p = a.parent[b0 + i];
  p = i > 0 && p >= 0 && p < i ? p : -1;
  const long long t = a.token64 ? ((const long long*)a.tokens)[b0 + i] : ((const int*)a.tokens)[b0 + i];
  const bool in = p >= 0 && t >= 0 && t < a.V;
  x = in ? (int)t : -1;
  px = in ? verify_value(((const T*)a.target)[(b0 + p) * a.t_row + t]) : 0.0;
  qx = !a.draft ? 1.0 : in ? verify_value(((const T*)a.draft)[(b0 + p) * a.d_row + t]) : 0.0;
}
__device__ __forceinline__ int verify_nodes(const VerifyArgs& a, int z, int& b0) {
  b0 = a.cu[z];
  const int b1 = a.cu[z + 1];
  return b0 >= 0 && b1 >= b0 && b1 <= a.T ? min(b1 - b0, TREE_NODES) : 0;
}

// The launch before the parts': every node's probabilities side by side, and the places of the sums
// empty.
template <typename T>
__device__ __forceinline__ void verify_gather_body(const VerifyArgs& a) {
  const int z = blockIdx.x;
  int b0;
  const int n = verify_nodes(a, z, b0);
  uint64_t* told = a.told + (long long)b0 * a.parts;
  for (int i = threadIdx.x; i < n * a.parts; i += 256) told[i] = VERIFY_EMPTY;
  for (int i = threadIdx.x; i < n; i += 256) {
    int p, x;
    verify_node<T>(a, b0, i, p, x, a.px[2 * (long long)(b0 + i)], a.px[2 * (long long)(b0 + i) + 1]);
  }
}

// PARTS: a.parts workgroups per sequence, behind verify_gather; else one.
template <typename T, bool PARTS>
__device__ __forceinline__ void verify_tree_body(const VerifyArgs& a) {
  using W = std::conditional_t<sizeof(T) == 4, verify_word4, verify_word2>;
  constexpr int N = 16 / (int)sizeof(T);
  __shared__ double px[TREE_NODES], qx[TREE_NODES];
  __shared__ float us[TREE_NODES];
  __shared__ int tok[TREE_NODES], gone[TREE_NODES];
  __shared__ short par[TREE_NODES];
  __shared__ double seg[2][VERIFY_WAVES], other[VERIFY_WAVES], scan[VERIFY_WAVES];
  __shared__ double upto[64];  // sum of the parts up to and with the one
  __shared__ unsigned long long missing;
  __shared__ int found, some;
  if (blockDim.x != VERIFY_THREADS) return;  // launch shape must match the kernel
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int parts = PARTS ? a.parts : 1;
  const int z = blockIdx.x / (unsigned)parts, part = blockIdx.x % (unsigned)parts;
  int b0;
  const int n = verify_nodes(a, z, b0);
  int* path = a.path + z * a.path_z;
  auto answer = [&](int token) {
    if (a.token64) ((long long*)a.next)[z * a.next_z] = token;
    else ((int*)a.next)[z * a.next_z] = token;
  };
  if (n == 0) {
    if (part) return;
    for (int i = tid; i < a.L; i += VERIFY_THREADS) path[i] = -1;
    if (tid == 0) {
      a.count[z * a.count_z] = 0;
      answer(-1);
    }
    return;
  }
  const T* P = (const T*)a.target;
  const T* Q = (const T*)a.draft;
  for (int i = tid; i < n; i += VERIFY_THREADS) {
    int p, x;
    if constexpr (PARTS) {
      p = a.parent[b0 + i];
      p = i > 0 && p >= 0 && p < i ? p : -1;
      const long long t = a.token64 ? ((const long long*)a.tokens)[b0 + i] : ((const int*)a.tokens)[b0 + i];
      x = p >= 0 && t >= 0 && t < a.V ? (int)t : -1;
      px[i] = a.px[2 * (long long)(b0 + i)];
      qx[i] = a.px[2 * (long long)(b0 + i) + 1];
    } else {
      verify_node<T>(a, b0, i, p, x, px[i], qx[i]);
    }
    par[i] = (short)p;
    tok[i] = x;
    us[i] = a.u[b0 + i];
  }
  __syncthreads();

  int cur = 0, count = 1, refused = 0, round = 0;
  double A = 0.0, S = 1.0, rest = 1.0;
  // N columns of a row from v on: near its end the last N, of which cover() says which are
  // columns v .. end - 1 (a row of fewer: element by element)
  auto place = [&](long long v) { return max(min(v, (long long)a.V - N), 0ll); };
  auto read = [&](const T* row, long long v) {
    if (a.V >= N) return u32x4(*(const W*)(row + place(v)));
    u32x4 w = {0, 0, 0, 0};
    for (int e = 0; e < a.V; ++e) {
      if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(row[e]);
      else w[e / 2] |= (uint32_t)row[e].bits << (16 * (e & 1));
    }
    return w;
  };
  auto cover = [&](long long v, long long end) {
    const int n = (int)max(min(end - v, (long long)N), 0ll);
    return n ? ((1u << n) - 1) << (int)(v - place(v)) : 0u;
  };
  // what is left of them
  auto left = [&](const u32x4& wp, const u32x4& wq, long long v, long long end, double (&r)[N]) {
    const uint32_t in = cover(v, end);
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = verify_element<T>(wp, e);
    // (A = 0 leaves p as it is, whatever q held: infinities too)
    if (Q && A > 0.0)
#pragma unroll
      for (int e = 0; e < N; ++e) r[e] = fmax(fma(-A, verify_element<T>(wq, e), r[e]), 0.0);
    if (!Q)
      for (int k = 0; k < refused; ++k) {
        const long long at = gone[k] - place(v);
#pragma unroll
        for (int e = 0; e < N; ++e) r[e] = at == e ? 0.0 : r[e];
      }
#pragma unroll
    for (int e = 0; e < N; ++e) r[e] = in >> e & 1 ? r[e] : 0.0;
  };
  // columns of a part, and of a wave of it: whole vectors
  const long long len = ((a.V + parts - 1) / parts + N - 1) / N * N;
  const long long share = ((len + VERIFY_WAVES - 1) / VERIFY_WAVES + N - 1) / N * N;
  auto bounds = [&](int of, int w, long long& from, long long& to) {
    const long long end = min((of + 1) * len, (long long)a.V);
    from = min(of * len + w * share, end);
    to = min(from + share, end);
  };
  // A wave's share of up to U vectors a lane of each row stays in registers: the next sum of the
  // same node and the search for the token need no loads.  (Longer shares are read again.)
  constexpr int U = 4;
  const bool fits = share <= 64 * N * U;
  u32x4 wp[U], wq[U];
  int held = -1;        // the node whose vectors they are
  bool held_q = false;  // q's as well
  // what is left of the node's row: S, and upto[] and seg[] as well.  (One place in the code
  // for all of it: code that runs a few times is bound by being fetched.)
  auto sum = [&]() {
    const T* pr = P + (long long)(b0 + cur) * a.t_row;
    const T* qr = Q + (long long)(b0 + cur) * a.d_row;
    const bool both = Q && A > 0.0;
    uint64_t todo = 1ull << part;
    bool alone = false;  // some sums were not told
    for (bool own = true; todo; own = false) {
      const int of = __ffsll((unsigned long long)todo) - 1;
      todo &= todo - 1;
      // the waves' sums of the part
      long long from, end;
      bounds(of, wave, from, end);
      if (!Q) __syncthreads();  // gone[]
      double t = 0.0;
      const bool here = own && held == cur && (held_q || !both);
#pragma unroll 1
      for (long long v0 = from + lane * N; v0 - lane * N < end; v0 += 64 * N * U) {
        if (!here)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            wp[u] = read(pr, v0 + 64 * N * u);
            wq[u] = both ? read(qr, v0 + 64 * N * u) : (u32x4){0, 0, 0, 0};
          }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (v0 - lane * N + 64 * N * u >= end) break;
          double r[N];
          left(wp[u], wq[u], v0 + 64 * N * u, end, r);
#pragma unroll
          for (int e = 0; e < N; ++e) t += r[e];
        }
      }
      held = own && fits ? cur : -1;
      held_q = here ? held_q : both;
      t = verify_lane(verify_scan(t), 63);
      if (!own) __syncthreads();  // (whoever read the sums before is done)
      if (lane == 0) (own ? seg[round & 1] : other)[wave] = t;
      __syncthreads();
      if (wave == 0) {
        t = 0.0;
#pragma unroll
        for (int w = 0; w < VERIFY_WAVES; ++w) t += (own ? seg[round & 1] : other)[w];
        if (!PARTS || !own) {
          if (lane == 0) upto[of] = t;
        } else {
          // told, and the others' taken
          uint64_t* told = a.told + (long long)(b0 + round) * parts;
          if (lane == 0)
            __hip_atomic_store(told + part, __builtin_bit_cast(uint64_t, t), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          bool have = lane == part || lane >= parts;
          t = lane < parts ? t : 0.0;
          // (the first look about when the others' sums can be there: looks before that are in their
          // way.  16 refusals in a row, one tree over 128000 columns, took 76 us without this wait, 56 with
          // it, 61 with one twice as long; with several looks on the way at a time 85)
          __builtin_amdgcn_s_sleep(15);
          for (int spin = 0; spin < VERIFY_SPINS && !__all(have); ++spin) {
            if (!have) {
              const uint64_t w = __hip_atomic_load(told + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
              have = w != VERIFY_EMPTY;
              if (have) t = __builtin_bit_cast(double, w);
            }
            __builtin_amdgcn_s_sleep(1);
          }
          const uint64_t none = __ballot(!have);
          if (none == 0) t = verify_scan(t);
          if (have && lane < parts) upto[lane] = t;
          if (lane == 0) missing = none;
        }
      }
      if (PARTS && own) {
        __syncthreads();
        todo = missing;
        alone = todo != 0;
      }
    }
    ++round;
    // (seg has two sides, so that a sum takes two barriers)
    if (!PARTS || alone) __syncthreads();
    if (PARTS && alone) {
      if (wave == 0) {
        const double t = verify_scan(lane < parts ? upto[lane] : 0.0);
        if (lane < parts) upto[lane] = t;
      }
      __syncthreads();
    }
    S = upto[parts - 1];
  };

  int at = 1;         // nodes before it are done with
  bool walk = true;   // the path goes on
  bool known = false; // S, seg and upto are those of this node with this A
  // the nodes of the window, one per lane
  int window = 0, up, mine_x, before = 0;  // before: refused children in earlier windows
  float mine_u;
  double mine_p, mine_q;
  uint64_t out = 0;  // the window's refused children
  auto load = [&]() {
    const int i = min(window + lane, n - 1);
    up = window + lane < n ? par[i] : -1;
    mine_x = tok[i];
    mine_u = us[i];
    mine_p = px[i];
    mine_q = qx[i];
    out = 0;
  };
  load();
  for (;;) {
    while (walk) {
      // the next child of the node: lane i holds node `window` + i, a test reads its lane
      uint64_t kids = 0;
      while (at < n && count < a.L) {
        if (at >= window + 64) {
          window = at & ~63;
          load();
          before = refused;
          __syncthreads();  // gone[]
        }
        kids = __ballot(up == cur) & (~0ull << (at - window));
        if (kids) break;
        at = window + 64;
      }
      if (!kids) {
        walk = false;
        break;
      }
      const int l = __ffsll((unsigned long long)kids) - 1;
      at = window + l + 1;
      const int x = __builtin_amdgcn_readlane(mine_x, l);
      const double p = verify_lane(mine_p, l), q = verify_lane(mine_q, l), u = (double)__builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine_u), l));
      double r = Q ? fmax(fma(-A, q, p), 0.0) : p;
      if (refused) {  // (without q: a token that was refused already is out)
        if (__ballot(mine_x == x) & out) r = 0.0;
        for (int k = 0; k < before; ++k) r = gone[k] == x ? 0.0 : r;
      }
      if (u * q * S < r * rest) {
        if (tid == 0 && part == 0) path[count] = window + l;
        ++count;
        cur = window + l;
        if (before) __syncthreads();  // gone[] has been read
        refused = before = 0;
        out = 0;
        A = 0.0;
        S = rest = 1.0;
        known = false;
      } else if (Q) {
        A += S / rest;
        if (a.distinct) rest = fmax(rest - q, 0x1p-24);
        known = false;
        break;
      } else {
        S -= r;
        if (tid == 0) gone[refused] = x;
        ++refused;
        out |= 1ull << l;
      }
    }
    if (!walk && known) {
      if (S > 0.0 || (A == 0.0 && refused == 0)) break;
      A = 0.0;  // nothing left: p itself
      refused = 0;
    }
    sum();
    known = true;
  }
  if (part == 0) {
    for (int i = count + tid; i < a.L; i += VERIFY_THREADS) path[i] = -1;
    if (tid == 0) {
      path[0] = 0;
      a.count[z * a.count_z] = count;
    }
  }
  // the first column whose sum passes the random number's share: its part (where none
  // does, the last with something left; part 0 of nothing), its wave, its column
  const double want = (double)a.last[z] * S;
  const double mine = upto[min(lane, parts - 1)], below = lane ? upto[min(lane, parts) - 1] : 0.0;
  const uint64_t over = __ballot(lane < parts && mine > want), some_left = __ballot(lane < parts && mine > below);
  const int of = over ? __ffsll((unsigned long long)over) - 1 : some_left ? 63 - __clzll((long long)some_left) : 0;
  if (of != part) return;
  double start = verify_lane(below, of);
  int w = 0;
  const double* waves = seg[(round - 1) & 1];
  while (w + 1 < VERIFY_WAVES && !(start + waves[w] > want)) start += waves[w++];
  while (w > 0 && !(waves[w] > 0.0)) start -= waves[--w];  // (a share past the end)
  long long from, end;
  bounds(part, w, from, end);
  if (held == cur) {  // the wave that has them
    if (wave != w) return;
    int some = -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long v = from + lane * N + 64 * N * u;
      if (v - lane * N >= end) break;
      double r[N], s = 0.0;
      left(wp[u], wq[u], v, end, r);
#pragma unroll
      for (int e = 0; e < N; ++e) s += r[e];
      const double t = verify_scan(s);
      double mine = start + (t - s);
      int hit = -1, any = -1;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        mine += r[e];
        if (r[e] > 0.0) {
          any = (int)(place(v) + e);
          if (hit < 0 && mine > want) hit = any;
        }
      }
      const uint64_t hits = __ballot(hit >= 0), anys = __ballot(any >= 0);
      if (hits) {
        if (lane == __ffsll((unsigned long long)hits) - 1) answer(hit);
        return;
      }
      if (anys) some = __builtin_amdgcn_readlane(any, 63 - __clzll((long long)anys));
      start += verify_lane(t, 63);
    }
    if (lane == 0) answer(max(some, 0));
    return;
  }
  const T* pr = P + (long long)(b0 + cur) * a.t_row;
  const T* qr = Q + (long long)(b0 + cur) * a.d_row;
  if (tid == 0) found = 0x7FFFFFFF, some = -1;
  __syncthreads();
  for (long long v0 = from; v0 < end; v0 += VERIFY_THREADS * N) {
    const long long v = v0 + tid * N;
    double r[N], s = 0.0;
    const u32x4 none = {0, 0, 0, 0};
    left(read(pr, v), Q && A > 0.0 ? read(qr, v) : none, v, end, r);
#pragma unroll
    for (int e = 0; e < N; ++e) s += r[e];
    const double t = verify_scan(s);
    if (lane == 63) scan[wave] = t;
    __syncthreads();
    double mine = start + (t - s);
#pragma unroll
    for (int k = 0; k < VERIFY_WAVES; ++k) mine += k < wave ? scan[k] : 0.0;
    int hit = -1, any = -1;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      mine += r[e];
      if (r[e] > 0.0) {
        any = (int)(place(v) + e);
        if (hit < 0 && mine > want) hit = any;
      }
    }
    if (hit >= 0) atomicMin(&found, hit);
    if (any >= 0) atomicMax(&some, any);
#pragma unroll
    for (int k = 0; k < VERIFY_WAVES; ++k) start += scan[k];
    __syncthreads();
    if (found != 0x7FFFFFFF) break;
  }
  if (tid == 0) answer(found != 0x7FFFFFFF ? found : some >= 0 ? some : 0);
}

}  // namespace g950

#define G950_VERIFY(TNAME, T)                                                                                     \
  extern "C" __global__ __launch_bounds__(256) void g950_verify_tree_##TNAME(const g950::VerifyArgs a) {        \
    g950::verify_tree_body<T, false>(a);                                                                          \
  }                                                                                                               \
  extern "C" __global__ __launch_bounds__(256) void g950_verify_tree_##TNAME##_parts(const g950::VerifyArgs a) { \
    g950::verify_tree_body<T, true>(a);                                                                           \
  }                                                                                                               \
  extern "C" __global__ __launch_bounds__(256) void g950_verify_tree_##TNAME##_gather(const g950::VerifyArgs a) { \
    g950::verify_gather_body<T>(a);                                                                               \
  }
G950_VERIFY(f32, float)
G950_VERIFY(bf16, g950::bf16_t)
G950_VERIFY(f16, g950::f16_t)
