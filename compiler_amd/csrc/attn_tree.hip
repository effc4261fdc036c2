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
  int base;       // keys before the tree; below 0: the first nodes have no cache row
};
__device__ __forceinline__ TreeSeq tree_seq(const int* cu, const int* used, int T, int most, int z) {
  TreeSeq s;
  const int b0 = cu[z], b1 = cu[z + 1];
  s.q0 = b0;
  s.n = b0 >= 0 && b1 >= b0 && b1 <= T ? b1 - b0 : 0;
  s.nq = min(s.n, most);
  s.base = max(max(used[z], 0) - s.n, -(1 << 20));  // (no node that takes part has a key below that)
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
// way from the node to its root meets them in order.  Not tuned: every (node, head) reads its keys
// by itself, each lane its own key's row value by value.  It is slower than the same formula in elementary torch
// calls but for one tree.  In ms, 32 heads on 8, this kernel / torch: 26 nodes over 1000 keys, 16 trees of 9 to 32 over 300
// to 4096, 32 single tokens over as many, 8 trees of 50 to 64 over 2049 to 8192
//   bfloat16, d 96             0.64 / 0.79    8.2 / 1.9   4.1 / 2.0   22.9 / 2.8
//   bfloat16, d 192            1.07 / 0.79   16.7 / 2.8   8.5 / 3.5   47.9 / 3.8
//   bfloat16, d 128, pages of 10 0.72 / 0.79 10.5 / 2.2   5.7 / 2.5   29.3 / 3.1
//   fp32, d 128                0.61 / 0.77    8.7 / 2.1   5.1 / 2.4   26.3 / 3.0
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

// ---------------------------------------------------------------- fast form
// bfloat16 and float16, d 64, 128 or 256, pages of whole 16-key runs, 16-byte rows.  A row is
// (node, head of the group).  A workgroup owns one (sequence, KV head, block of 32 RW
// rows, key range); its 4 waves are RW blocks of 32 rows times KW = 4 / RW shares of the
// keys, so that K and V are read once for all rows of a block, whatever their number.
//   * S^T = K.Q^T on v_mfma_f32_32x32x16: a lane holds 16 of 32 keys' scores of ONE row, so
//     the softmax's running maximum and sum are per lane (two lanes a row).  Its keys 4 g .. + 3
//     and 8 + 4 g .. + 3 of every 16 are the contraction slots that its own probabilities
//     feed in O^T = V^T.P^T; V^T's fragments of the same keys come from transposing LDS reads.
//   * K and V come by direct global->LDS DMA into a ring of stages, TKS keys each, K two
//     stages ahead and V one (d 256: both one).  16-byte pieces are swizzled on the way (the source address is the
//     lane's): K's by the key, so that the 16 keys of a read lie in all 64 banks, V's
//     by 64 bytes, so that the four keys of a transposing read do.
//   * Stages are taken from the last to the first: the tree's keys come first, and a lane
//     meets the nodes above its own one as it walks to the root, parents from LDS;
//     each 32-key tile of the tree costs it a word of visible keys.  Tiles that every row
//     sees whole (all but a few) skip that.
//   * What a row does not see may hold anything: scores are replaced, and where V of a
//     stage that some row does not see whole is not finite, 0 V would not be 0: such values
//     are added, key by key, where a row sees them, and taken out of the stage.
//   * A probability is rounded to the operands' type, once, for P.V (half a step of itself; the sum l and O
//     stay in fp32): exact products would take a second 16-bit term and P.V's MFMAs twice.  O's
//     distance from the formula's is 0.0023 of it in bfloat16 (root mean squares; 0.0017 of that
//     is the rounding of O), 0.00028 in float16 (0.0002).
// Bound by K and V for few rows, by the matrix cores and the softmax's vector ALU from 64 rows
// on, and for short batches by a start of some 8 us (dealing the keys 1.6, queries, parents and
// page table 1.8, the first K 1.9, its scores and the way up the tree 2.3) with 3 behind the last
// stage.  32 heads on 8 in bfloat16, parts + joining: 32 single tokens over 300 to 4096 keys
// 64 + 5.3 us at d 128 (4.5 TB/s), 38 + 5 at 64, 140 + 6.4 at 256; 16 trees of 9 to 32 nodes over as many 42 + 10, 23 + 6,
// 95 + 17; 8 of 50 to 64 over 2049 to 8192 61 + 11 (39 GFLOP) at d 128, 178 + 18 at 256; 64 trees of 32 over
// 8192 390 in all (5.5 TB/s), of 64 565 to 640 (0.86 to 0.97 PFLOP/s).  The way up is walked node by node: one
// chain of 64 nodes over 4096 keys 32 where as many children of one root take 29, of 1024 149 and 100; 16 chains
// of 1024 1320 and 1100.  512 threads a workgroup, halves taking turns on the matrix cores: 52 to 58 in
// place of 43, 780 to 880 in place of 540 to 730.

struct TreeSpan {
  TreeSeq sq;
  int kend;     // keys past the last that can be seen
  int kbeg, n;  // tiles of 64 keys from kbeg on; 0 where no node takes part, else at least 1
};
__device__ __forceinline__ TreeSpan tree_span(const AttnTreeArgs& p, int z) {
  TreeSpan s;
  s.sq = tree_seq(p.cu, p.used, p.T, p.seqlen_q, z);
  const long long held = p.pages > 0 ? (long long)p.max_pages * p.block_size : 0;
  s.kend = (int)min((long long)max(s.sq.base + s.sq.nq, 0), held);
  s.kbeg = p.left < 0 ? 0 : max(0ll, (long long)s.sq.base - p.left) / 64 * 64;
  s.n = s.sq.nq > 0 ? max(1, (s.kend - s.kbeg + 63) / 64) : 0;
  return s;
}

// sums of `v` over the lanes up to the own one
__device__ __forceinline__ int tree_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return v;
}

// How the batch's keys are dealt: every sequence's tiles are cut into parts of c (the last
// one shorter), c so that all sequences together have at most p.parts parts.  The lengths
// live on the device, so each wave works this out, 64 sequences at a time: a batch of different lengths becomes parts of one length, and as
// many as the chip has places for.
struct TreeDeal {
  const AttnTreeArgs& p;
  int n0;  // tiles of sequence `lane`, the first 64 of the batch
  int c;
  __device__ __forceinline__ int tiles(int z0) const {
    const int z = z0 + (int)(threadIdx.x & 63);
    return z < p.B ? tree_span(p, z).n : 0;
  }
  __device__ __forceinline__ int tiles_again(int z0) const { return z0 ? tiles(z0) : n0; }
  __device__ __forceinline__ explicit TreeDeal(const AttnTreeArgs& args) : p(args) {
    n0 = tiles(0);
    long long sum = 0;
    for (int z0 = 0; z0 < p.B; z0 += 64) {
      const int n = tiles_again(z0);
      sum += __builtin_amdgcn_readlane(tree_scan(n), 63);
    }
    // the least c that gives no more than p.parts: between those of parts without remainders and
    // with one for every sequence
    // (no sequence has more than 2^25 tiles)
    int lo = max((int)min((sum + p.parts - 1) / p.parts, 1ll << 25), p.min_tiles);
    c = max((int)min((sum + p.parts - p.B - 1) / (p.parts - p.B), 1ll << 25), p.min_tiles);
    while (lo < c) {
      const int mid = (uint32_t)(lo + c) / 2;
      int n = 0;
      for (int z0 = 0; z0 < p.B; z0 += 64) n += __builtin_amdgcn_readlane(tree_scan(cut(tiles_again(z0), mid)), 63);
      if (n <= p.parts) c = mid;
      else lo = mid + 1;
    }
  }
  static __device__ __forceinline__ int cut(int n, int c) { return (uint32_t)(n + c - 1) / (uint32_t)c; }
  // the sequence that part `part` belongs to, and the parts before that sequence; -1: none
  __device__ __forceinline__ int sequence(int part, int& before) const {
    int start = 0;
    for (int z0 = 0; z0 < p.B; z0 += 64) {
      const int k = cut(tiles_again(z0), c), upto = start + tree_scan(k);
      const uint64_t past = __ballot(upto > part);
      if (past) {
        const int at = __ffsll((unsigned long long)past) - 1;
        before = __builtin_amdgcn_readlane(upto - k, at);
        return z0 + at;
      }
      start = __builtin_amdgcn_readlane(upto, 63);
    }
    return -1;
  }
  // the parts before sequence z
  __device__ __forceinline__ int before(int z) const {
    int start = 0;
    for (int z0 = 0;; z0 += 64) {
      const int k = cut(tiles_again(z0), c), upto = start + tree_scan(k);
      if (z < z0 + 64) return __builtin_amdgcn_readlane(upto - k, z - z0);
      start = __builtin_amdgcn_readlane(upto, 63);
    }
  }
};

// What a workgroup does: tiles t0 .. t1 - 1 of a block of rows of a (sequence, KV head); rec:
// where its partial rows go, -1 if it has all the tiles.  Blocks and heads of a part are neighbours:
// the blocks, which read the same keys, are a multiple of 8 apart where there are 8 heads, so that one
// XCD's L2 has them.
struct TreePart {
  int z, hk, block, t0, t1, rec;
};
__device__ __forceinline__ TreePart tree_deal(const AttnTreeArgs& p, TreeSpan& sp) {
  const uint32_t heads = p.Hkv, units = heads * p.row_blocks, unit = blockIdx.x % units;
  const int part = blockIdx.x / units;
  TreePart w;
  w.hk = unit % heads;
  w.block = unit / heads;
  w.t0 = 0;
  w.rec = -1;
  if (p.parts == 0) {
    w.z = part;
    sp = tree_span(p, w.z);
    w.t1 = sp.n;
    return w;
  }
  const TreeDeal d(p);
  int before = 0;
  w.z = d.sequence(part, before);
  if (w.z < 0) {
    sp.n = 0;
    return w;
  }
  sp = tree_span(p, w.z);
  w.t0 = (part - before) * d.c;
  w.t1 = min(sp.n, w.t0 + d.c);
  if (sp.n > d.c) w.rec = blockIdx.x;
  return w;
}

// value of `v` combined over the two lanes holding one row
template <class Op>
__device__ __forceinline__ float tree_row(float v) {
  return Op::apply(v, __shfl_xor(v, 32));
}

__device__ __forceinline__ void tree_barrier() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// a value of the type (low half) that is not finite and `sees`, else 0
template <bool F16>
__device__ __forceinline__ float tree_odd(uint32_t w, bool sees) {
  constexpr uint32_t EXP = F16 ? 0x7C00u : 0x7F80u;
  const float x = F16 ? f16_to_f32((uint16_t)w) : bf16_to_f32((uint16_t)w);
  return sees && (w & EXP) == EXP ? x : 0.0f;
}
template <bool F16>
__device__ __forceinline__ uint32_t tree_finite(uint32_t w) {
  constexpr uint32_t EXP = F16 ? 0x7C00u : 0x7F80u;
  if ((w & EXP) == EXP) w &= 0xFFFF0000u;
  if ((w >> 16 & EXP) == EXP) w &= 0xFFFFu;
  return w;
}
template <int D, int RW>
struct TreeCfg {
  static constexpr int KW = 4 / RW;
  static constexpr int SUB = KW == 1 ? 2 : 1;           // 32-key tiles of a wave in a stage
  static constexpr int TKS = 32 * KW * SUB;             // keys of a stage: 64
  static constexpr int ROW = 2 * D, KT = TKS * ROW, STAGE = 2 * KT;
  static constexpr int ROWS = 32 * RW;
  static constexpr int LDS = 2 * STAGE;
  static_assert(LDS >= 4 * 32 * D * 4, "the waves' partial O fits the ring");
};

template <int D, bool F16, int RW>
__device__ __forceinline__ void attn_tree_body(const AttnTreeArgs& p) {
  using C = TreeCfg<D, RW>;
  constexpr int KW = C::KW, SUB = C::SUB, TKS = C::TKS, ROW = C::ROW, KT = C::KT, ROWS = C::ROWS;
  constexpr int KPI = 1024 / ROW, CH = ROW / 16;  // keys of a DMA instruction, 16-byte pieces of a row
  constexpr int DI = 16 / KPI;                    // DMA instructions of 16 keys' K
  constexpr int RUNS = TKS / 16, RPW = RUNS / 4;  // 16-key runs of a stage, of a wave's loads
  constexpr int SB = 64 / RUNS;                   // stages of which the lanes hold the runs' pages
  constexpr int DS = D / 16, DB = D / 32;
  __shared__ __attribute__((aligned(1024))) char lds[C::LDS];
  __shared__ short par[TREE_NODES];
  __shared__ float ml[4][32][2];
  __shared__ int odd[4];
  __shared__ float share[ROWS][KW];
  __shared__ long long place[ROWS];
  if (blockDim.x != 256) return;  // launch shape must match the kernel
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = wave / KW, kw = wave % KW;
  const int g = lane >> 5, r32 = lane & 31;
  const uint32_t G = p.group;
  TreeSpan sp;
  const TreePart w = tree_deal(p, sp);
  const TreeSeq& sq = sp.sq;
  const int rows = sq.nq * p.group, row0 = w.block * ROWS;
  if (row0 >= rows || w.t0 >= sp.n) return;
  const int nrows = min(ROWS, rows - row0);
  const bool busy = rw * 32 < nrows;
  const int lo = sp.kbeg + 64 * w.t0, hi = min(sp.kend, sp.kbeg + 64 * w.t1);
  const int nst = hi > lo ? (hi - lo + TKS - 1) / TKS : 0;

  // this lane's row: its node, its query
  const uint32_t row = row0 + min(rw * 32 + r32, nrows - 1);
  const int node = row / G;
  u32x4 qf[DS];
  {
    const char* src = (const char*)p.q + 2 * ((long long)(sq.q0 + node) * p.q_st + (long long)(w.hk * G + row % G) * p.q_sh + 8 * g);
#pragma unroll
    for (int ks = 0; ks < DS; ++ks) qf[ks] = *(const u32x4*)(src + 32 * ks);
  }
  const bool tree = hi > sq.base || p.left >= 0;
  if (tree)
    for (int i = tid; i < sq.nq; i += 256) par[i] = (short)tree_parent(p.parent, sq, i);

  const uint32_t ring32 = lds_addr(lds);
  const char* kbase = (const char*)p.k + 2 * (long long)w.hk * p.k_h;
  const char* vbase = (const char*)p.v + 2 * (long long)w.hk * p.v_h;
  auto kswz = [](int key) { return D == 64 ? (key >> 1) & 7 : key & 15; };
  auto vswz = [](int key) { return D == 64 ? (key >> 1) & 1 : key & 3; };
  const uint32_t k_r = 2 * (uint32_t)p.k_r, v_r = 2 * (uint32_t)p.v_r;
  const int dkey = lane / CH, dpos = lane % CH;
  uint32_t koff[DI], voff[DI];
#pragma unroll
  for (int u = 0; u < DI; ++u) {
    const int key = u * KPI + dkey;
    koff[u] = key * k_r + ((dpos ^ kswz(key)) << 4);
    voff[u] = key * v_r + ((dpos ^ (vswz(key) << 2)) << 4);
  }
  // pages and rows of the runs of SB stages, one per lane, looked up a stage before they are
  // needed; a run without a page (or past the end) reads page 0 and is masked
  const int* table = p.table + (long long)w.z * p.table_s;
  int next = -1, pages = 0, prow = 0;
  uint64_t live[2] = {0, 0};  // by the parity of the batch of SB stages
  auto batch_key = [&](int j) { return lo + TKS * (nst - 1 - (j + lane / RUNS)) + 16 * (lane % RUNS); };
  auto look = [&](int j) {
    const int key = batch_key(j), e = (uint32_t)max(key, 0) / (uint32_t)p.block_size;
    next = key >= lo && key < hi && e < p.max_pages ? table[e] : -1;
  };
  uint32_t pg[RPW], pr[RPW];  // of the wave's runs of the last stage whose K was issued
  auto stage_pages = [&](int j) {
    if (j % SB == 0) {
      const int key = batch_key(j), ph = next < p.pages ? next : -1;
      const uint64_t m = __ballot(ph >= 0);
      if ((j / SB) & 1) live[1] = m;
      else live[0] = m;
      pages = max(ph, 0);
      prow = ph < 0 ? 0 : (uint32_t)key % (uint32_t)p.block_size;
    }
#pragma unroll
    for (int x = 0; x < RPW; ++x) {
      const int at = j % SB * RUNS + wave + 4 * x;
      pg[x] = __builtin_amdgcn_readlane(pages, at);
      pr[x] = __builtin_amdgcn_readlane(prow, at);
    }
  };
  auto dma = [&](const char* base, long long page, uint32_t step, const uint32_t (&off)[DI], uint32_t dst) {
#pragma unroll
    for (int x = 0; x < RPW; ++x) {
      const char* src = base + 2 * (pg[x] * (uint64_t)page) + (uint64_t)pr[x] * step;
#pragma unroll
      for (int u = 0; u < DI; ++u) dma_base16(src, off[u], dst + (wave + 4 * x) * 16 * ROW + u * 1024);
    }
  };
  auto dma_k = [&](uint32_t dst) { dma(kbase, p.k_p, k_r, koff, ring32 + dst); };
  auto dma_v = [&](uint32_t dst) { dma(vbase, p.v_p, v_r, voff, ring32 + dst); };

  // (the queries are waited for here, not by the compiler's count in the loop, where it
  // would take the DMA's loads along)
#pragma unroll
  for (int ks = 0; ks < DS; ++ks) asm volatile("" : "+v"(qf[ks]));
  look(0);
  __syncthreads();  // parents
  int first = 0;    // first key before the tree that the row sees
  if (p.left >= 0) {
    int depth = 0;
    for (int c = par[node]; c >= 0; c = par[c]) ++depth;
    first = max(0ll, (long long)sq.base + depth - p.left);
  }
  int cur = node, up = 0;  // next node of the way to the root, levels above the own

  f32x16 o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[b][e] = 0.0f;
  float ms = -__builtin_huge_valf(), l[4] = {};
  const float c2 = p.scale_log2;
  // operand reads: K of key r32, V of keys 4 g + (lane & 15) / 4 .. of a 16-d half block
  const int kread = r32 * ROW, kx = (g ^ kswz(r32)) << 4;
  const int j16 = lane & 15;
  const int vread = (4 * g + (j16 >> 2)) * ROW + 32 * ((lane >> 4) & 1) + 8 * (j16 & 3), vx = vswz(j16 >> 2) << 6;
  const uint32_t own = kw * 32 * SUB * ROW;  // this wave's keys of a stage
  f32x16 s[SUB];
  u32x4 pf[SUB][2];
  uint32_t vis[SUB];  // the row's visible keys of each tile of a masked stage
  // S^T of a wave's tiles (K at `kp`)
  auto scores = [&](const char* kp) {
#pragma unroll
    for (int t = 0; t < SUB; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[t][e] = 0.0f;
#pragma unroll
    for (int ks = 0; ks < DS; ++ks)
#pragma unroll
      for (int t = 0; t < SUB; ++t)
        s[t] = mfma16<F16>(*(const u32x4*)(kp + t * 32 * ROW + kread + (kx ^ (ks << 5))), qf[ks], s[t]);
  };
  // stage i's scores of unseen keys replaced
  auto mask = [&](int i) {
    const int kv0 = lo + TKS * (nst - 1 - i) + 32 * SUB * kw;
    const uint32_t alive = (uint32_t)(live[(i / SB) & 1] >> (i % SB * RUNS + 2 * SUB * kw)) & ((1u << (2 * SUB)) - 1);
#pragma unroll
    for (int t = 0; t < SUB; ++t) vis[t] = ~0u;
    if (alive == (1u << (2 * SUB)) - 1 && kv0 + 32 * SUB <= min(sq.base, hi) && !__any(first > kv0)) return;
#pragma unroll
    for (int t = SUB - 1; t >= 0; --t) {
      const int k0 = kv0 + 32 * t, n0 = k0 - sq.base;  // first key, and as a node
      uint32_t v = n0 <= -32 ? ~0u : n0 < 0 ? (1u << -n0) - 1 : 0u;
      if (first > k0) v &= first - k0 < 32 ? ~0u << (first - k0) : 0u;
      // (nodes behind the range are walked by the part that they belong to, or have no cache
      // row: here there may be no parents)
      if (n0 > -32 && k0 < hi && hi > sq.base)
        while (cur >= max(n0, 0)) {
          if (cur - n0 < 32 && (p.left < 0 || up <= p.left)) v |= 1u << (cur - n0);
          cur = par[cur];
          ++up;
        }
      if (hi - k0 < 32) v &= hi > k0 ? (1u << (hi - k0)) - 1 : 0u;
      if (!(alive >> (2 * t) & 1)) v &= 0xFFFF0000u;
      if (!(alive >> (2 * t + 1) & 1)) v &= 0xFFFFu;
      vis[t] = v;
      v >>= 4 * g;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!(v >> (8 * (e >> 2) + (e & 3)) & 1)) s[t][e] = -__builtin_huge_valf();
    }
  };
  auto softmax = [&]() {
    float mh = s[0][0];
#pragma unroll
    for (int t = 0; t < SUB; ++t)
#pragma unroll
      for (int e = 0; e < 16; e += 2) mh = vmax3(mh, s[t][e], s[t][e + 1]);
    mh *= c2;
    if (__any(mh > ms + 8.0f)) {
      const float mt = tree_row<OpMax>(mh);
      const bool move = mt > ms + 8.0f;
      const float alpha = move ? __builtin_amdgcn_exp2f(ms - mt) : 1.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) l[e] *= alpha;
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] *= alpha;
      ms = move ? mt : ms;
    }
    // rows without a visible key so far: exponent base 0, exp2(-inf) = 0
    const float mb = ms == -__builtin_huge_valf() ? 0.0f : ms;
#pragma unroll
    for (int t = 0; t < SUB; ++t) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        s[t][e] = __builtin_amdgcn_exp2f(fmaf(s[t][e], c2, -mb));
        l[e & 3] += s[t][e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) pf[t][e >> 2][e & 3] = pack2(s[t][2 * e], s[t][2 * e + 1], F16);
    }
  };
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  auto vfrag = [&](const char* vp, int t, int k2, int b) {
    u32x4 f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(vp + (32 * t + 16 * k2 + 8 * h) * ROW + vread + ((b << 6) ^ vx))));
      f[2 * h] = x[0];
      f[2 * h + 1] = x[1];
    }
    return f;
  };
  // O^T += V^T.P^T of a wave's tiles (V at `vp`)
  auto values = [&](const char* vp) {
#pragma unroll
    for (int t = 0; t < SUB; ++t)
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int b = 0; b < DB; ++b) o[b] = mfma16<F16>(vfrag(vp, t, k2, b), pf[t][k2], o[b]);
  };
  // Stage i (V at `vp`) where some row does not see all of it: what is not finite in V is
  // added to the rows that see it and taken out of the tile.  Called by all waves, behind the
  // softmax.
  auto clean = [&](int i, char* vp) {
    const int kv0 = lo + TKS * (nst - 1 - i);
    const uint32_t alive = (uint32_t)(live[(i / SB) & 1] >> (i % SB * RUNS)) & ((1u << RUNS) - 1);
    if (alive == (1u << RUNS) - 1 && kv0 + TKS <= min(sq.base, hi) && (p.left < 0 || (long long)sq.base + sq.nq - p.left <= kv0)) return;
    // an exponent of ones carries into the bit above it
    constexpr uint32_t EXP = F16 ? 0x7C007C00u : 0x7F807F80u, CARRY = F16 ? 0x04000400u : 0x00800080u;
    uint32_t found = 0;
#pragma unroll 4
    for (int x = tid; x < KT / 16; x += 256) {
      const u32x4 f = *(const u32x4*)(vp + x * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) found |= (f[e] & EXP) + CARRY;
    }
    found = __any(found & 0x80008000u);
    if (lane == 0) odd[wave] = (int)found;
    __syncthreads();
    if (!(odd[0] | odd[1] | odd[2] | odd[3])) return;
    if (busy)
#pragma unroll
      for (int t = 0; t < SUB; ++t)
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {  // this lane's dims 32 b + 8 e + 4 g .. + 3 of the key
          const bool sees = vis[t] >> k & 1;
#pragma unroll
          for (int b = 0; b < DB; ++b) {
            __builtin_amdgcn_sched_barrier(0);  // (a few values at a time)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const u32x2 x = *(const u32x2*)(vp + (32 * (kw * SUB + t) + k) * ROW + ((b ^ vswz(k)) << 6) + 16 * e + 8 * g);
#pragma unroll
              for (int h = 0; h < 4; ++h) o[b][4 * e + h] += tree_odd<F16>(x[h >> 1] >> (16 * (h & 1)), sees);
            }
          }
        }
    __syncthreads();
#pragma unroll 1
    for (int x = tid; x < KT / 16; x += 256) {
      u32x4 f = *(const u32x4*)(vp + x * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = tree_finite<F16>(f[e]);
      *(u32x4*)(vp + x * 16) = f;
    }
    __syncthreads();
  };

  if constexpr (D < 256) {
    // Bound by the matrix cores and the vector ALU beside the bytes.  Iteration i: V of
    // stage i and K of i + 1 have landed; softmax of stage i, then its V and the next
    // stage's scores in one run of MFMAs at raised priority, whose operand reads are issued ahead
    // of them (two groups of V, eight fragments of K): the softmax of one of the two
    // waves of a SIMD runs beside the MFMAs of the other.  K is issued two stages ahead, V one.
    auto kat = [&](int i) { return (uint32_t)(i & 1) * KT; };
    auto vat = [&](int i) { return (uint32_t)(2 + (i & 1)) * KT; };
    constexpr int R = 2 * DB, NV = 2 * SUB, NK = SUB * DS;
    u32x2 vt[2][R];
    u32x4 kf[8];
    auto vread_ = [&](auto ic, uint32_t slot) {  // group I: V of keys 16 I .. + 15
      constexpr int I = decltype(ic)::value;
      static_for<R>([&](auto qc) {
        constexpr int Q = decltype(qc)::value;
        lds_rdtr<(16 * I + 8 * (Q & 1)) * ROW>(vt[I & 1][Q], ring32 + slot + own + vread + (((Q >> 1) << 6) ^ vx));
      });
    };
    auto vmma = [&](auto ic) {
      constexpr int I = decltype(ic)::value;
      static_for<DB>([&](auto bc) {
        constexpr int B = decltype(bc)::value;
        const u32x4 vf = {vt[I & 1][2 * B][0], vt[I & 1][2 * B][1], vt[I & 1][2 * B + 1][0], vt[I & 1][2 * B + 1][1]};
        o[B] = mfma16<F16>(vf, pf[I >> 1][I & 1], o[B]);
      });
    };
    auto kread_ = [&](auto jc, uint32_t slot) {  // fragment J: tile J % SUB, k-step J / SUB
      constexpr int J = decltype(jc)::value;
      if constexpr (J < NK)
        lds_rd128<(J % SUB) * 32 * ROW>(kf[J & 7], ring32 + slot + own + kread + (kx ^ ((J / SUB) << 5)));
    };
    auto kahead = [&](uint32_t slot) { static_for<4>([&](auto jc) { kread_(jc, slot); }); };
    // O^T += V^T.P^T, with the first four fragments of the next K on the way (each wait
    // names how many reads were issued after the group it completes).  What is read ahead is
    // waited for in the same run of code: no branch or copy meets a register in flight.
    auto run_v = [&](uint32_t vslot, uint32_t kslot) {
      vread_(std::integral_constant<int, 0>{}, vslot);
      vread_(std::integral_constant<int, 1>{}, vslot);
      static_for<NV>([&](auto ic) {
        constexpr int I = decltype(ic)::value;
        if constexpr (I + 1 == NV) kahead(kslot);
        constexpr int after = I + 1 < NV ? R : 4;
        lds_wait<after>(vt[I & 1]);
        vmma(ic);
        if constexpr (I + 2 < NV) vread_(std::integral_constant<int, I + 2>{}, vslot);
      });
    };
    auto run_k = [&](uint32_t slot) {
      static_for<4>([&](auto jc) { kread_(std::integral_constant<int, decltype(jc)::value + 4>{}, slot); });
      static_for<NK>([&](auto jc) {
        constexpr int J = decltype(jc)::value;
        constexpr int after = NK - J - 1 < 7 ? NK - J - 1 : 7;
        lds_wait<after>(kf[J & 7]);
        s[J % SUB] = mfma16<F16>(kf[J & 7], qf[J / SUB], J < SUB ? (f32x16){} : s[J % SUB]);
        kread_(std::integral_constant<int, J + 8>{}, slot);
      });
    };
    if (nst > 0) {
      stage_pages(0);
      dma_k(kat(0));
      dma_v(vat(0));
    }
    if (nst > 1) {
      stage_pages(1);
      dma_k(kat(1));
    }
    // K of stage 0 has landed (V of stage 0 and K of stage 1 may be in flight)
    if (nst > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * DI * RPW) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(DI * RPW) : "memory");
    tree_barrier();
    if (busy && nst > 0) {
      kahead(kat(0));
      run_k(kat(0));
    }
    for (int i = 0; i < nst; ++i) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      tree_barrier();
      // (into the slots of K of stage i, whose scores are formed, and of V of stage i - 1)
      if (i + 1 < nst) dma_v(vat(i + 1));
      if (i + 2 < nst) {
        stage_pages(i + 2);
        dma_k(kat(i + 2));
        if ((i + 3) % SB == 0) look(i + 3);
      }
      if (busy) {
        mask(i);
        softmax();
      }
      clean(i, lds + vat(i));
      if (busy) {
        __builtin_amdgcn_s_setprio(2);
        // (behind the last stage the scores are those of what the slot holds, and nobody's)
        run_v(vat(i), kat(i + 1));
        run_k(kat(i + 1));
        __builtin_amdgcn_s_setprio(0);
      }
    }
    tree_barrier();
  } else {
    // (no registers for reads ahead: whole stages, products as the compiler orders them)
    auto issue = [&](int j) {
      stage_pages(j);
      dma_k((j & 1) * C::STAGE);
      dma_v((j & 1) * C::STAGE + KT);
      if ((j + 1) % SB == 0) look(j + 1);
    };
    if (nst > 0) issue(0);
    if (nst > 1) issue(1);
    for (int i = 0; i < nst; ++i) {
      // stage i has landed once at most the next one's loads are in flight
      if (i + 1 < nst) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * RPW * DI) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      tree_barrier();
      char* st = lds + (i & 1) * C::STAGE;
      if (busy) {
        scores(st + own);
        mask(i);
        softmax();
      }
      clean(i, st + KT);
      if (busy) values(st + KT + own);
      // every wave's LDS reads have returned before the stage's slot is refilled
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      tree_barrier();
      if (i + 2 < nst) issue(i + 2);
    }
  }

  // ---- the waves' partial rows through the ring (16-byte pieces XOR-swizzled by the row),
  // maxima and sums beside it
  char* mine = lds + wave * 32 * D * 4;
  const float ls = tree_row<OpSum>((l[0] + l[1]) + (l[2] + l[3]));
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *(f32x4*)(mine + r32 * D * 4 + (((8 * b + 2 * e + g) ^ (r32 & 15)) << 4)) =
          (f32x4){o[b][4 * e], o[b][4 * e + 1], o[b][4 * e + 2], o[b][4 * e + 3]};
  if (g == 0) {
    ml[wave][r32][0] = ms;
    ml[wave][r32][1] = ls;
  }
  __syncthreads();
  // a row's weights of its waves' shares and its place: worked out once for all of its pieces
  if (tid < nrows) {
    const int w0 = tid / 32 * KW, rr = tid % 32;
    float m = ml[w0][rr][0], lt = 0.0f, f[KW];
#pragma unroll
    for (int x = 1; x < KW; ++x) m = fmaxf(m, ml[w0 + x][rr][0]);
#pragma unroll
    for (int x = 0; x < KW; ++x) {
      // no finite score: no key of this row (l = 0), or only NaN ones
      f[x] = ml[w0 + x][rr][0] == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(ml[w0 + x][rr][0] - m);
      lt = fmaf(f[x], ml[w0 + x][rr][1], lt);
    }
    const bool empty = !(lt > 0.0f);  // zero or NaN
    const uint32_t at = row0 + tid, i = at / G, h = w.hk * G + at % G;
    if (w.rec >= 0) {
      const long long rec = (long long)w.rec * p.merge_rows + tid;
      *(f32x2*)(p.ml + 2 * rec) = (f32x2){m, lt};
      place[tid] = rec * D;
    } else {
      p.lse[(long long)h * p.lse_h + (long long)(sq.q0 + i) * p.lse_t] =
          empty ? __builtin_huge_valf() : (m + __log2f(lt)) * 0.69314718055994530942f;
      place[tid] = (long long)(sq.q0 + i) * p.o_st + (long long)h * p.o_sh;
    }
#pragma unroll
    for (int x = 0; x < KW; ++x) share[tid][x] = w.rec >= 0 || empty ? f[x] : f[x] / lt;
  }
  __syncthreads();
  constexpr int CPR = D / 4;  // 16-byte pieces (4 d) of a row
#pragma unroll 4
  for (int k = 0; k < ROWS * CPR / 256; ++k) {
    const int r = (tid + 256 * k) / CPR, c = tid % CPR, w0 = r / 32 * KW, rr = r % 32;
    if (r >= nrows) break;
    f32x4 sum = {};
#pragma unroll
    for (int x = 0; x < KW; ++x) {
      const f32x4 ow = *(const f32x4*)(lds + (w0 + x) * 32 * D * 4 + rr * D * 4 + ((c ^ (rr & 15)) << 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(share[r][x], ow[e], sum[e]);
    }
    if (w.rec >= 0) *(f32x4*)(p.part + place[r] + c * 4) = sum;
    else *(u32x2*)((uint16_t*)p.o + place[r] + c * 4) = (u32x2){pack2(sum[0], sum[1], F16), pack2(sum[2], sum[3], F16)};
  }
}

// Joins the parts of a block of rows, 16 bytes of a row per lane, U parts at a time: NW
// waves per 256 / D rows, which take the parts in turn.
template <int D, bool F16, int ROWS, int NW>
__device__ __forceinline__ void attn_tree_merge_body(const AttnTreeArgs& p) {
  constexpr int LPR = D / 4, AT = 64 / LPR, U = 8;  // lanes of a row, rows of a wave
  __shared__ float js[NW][64][6];
  if (blockDim.x != (NW == 1 ? 256 : 64 * NW)) return;  // launch shape must match the kernel
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int nw = NW;
  const int share = NW == 1 ? 0 : wave;
  const uint32_t item = NW == 1 ? blockIdx.x * 4 + wave : blockIdx.x, groups = (p.merge_rows + AT - 1) / AT;
  const uint32_t id = item / groups, r0 = item % groups * AT;
  const uint32_t heads = p.Hkv, units = heads * p.row_blocks, unit = id % units;
  const int z = id / units, hk = unit % heads, block = unit / heads;
  if (z >= p.B) return;
  const TreeDeal d(p);
  const TreeSpan sp = tree_span(p, z);
  const int rows = min(sp.sq.nq * p.group - block * ROWS, ROWS), count = (sp.n + d.c - 1) / d.c;
  if ((int)r0 >= rows || count <= 1) return;  // (one part: its workgroup had all of it)
  const int r = min((int)r0 + lane / LPR, rows - 1);
  const long long rec = ((long long)d.before(z) * units + unit) * p.merge_rows + r, step = (long long)units * p.merge_rows;
  const float* part = p.part + rec * D + lane % LPR * 4;
  const float* pair = p.ml + 2 * rec;
  float m = -__builtin_huge_valf(), l = 0.0f;
  f32x4 acc = {};
  for (int s0 = share; s0 < count; s0 += U * nw) {
    f32x4 v[U];
    f32x2 ml[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long s = min(s0 + u * nw, count - 1) * step;
      v[u] = *(const f32x4*)(part + s * D);
      ml[u] = *(const f32x2*)(pair + s * 2);
    }
    float to = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * nw < count) to = fmaxf(to, ml[u][0]);
    // no finite score so far, or in a part: nothing seen (O = l = 0), or only NaN, which stays
    const float was = m == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(m - to);
    acc *= was;
    l *= was;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u * nw < count) {
        const float f = ml[u][0] == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(ml[u][0] - to);
        l = fmaf(f, ml[u][1], l);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, v[u][e], acc[e]);
      }
    m = to;
  }
  if constexpr (NW > 1) {
    float* mine = js[wave][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) mine[e] = acc[e];
    mine[4] = m;
    mine[5] = l;
    __syncthreads();
    if (wave) return;
    float to = m;
#pragma unroll
    for (int w = 1; w < NW; ++w) to = fmaxf(to, js[w][lane][4]);
    acc = (f32x4){};
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float* x = js[w][lane];
      const float f = x[4] == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(x[4] - to);
      l = fmaf(f, x[5], l);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, x[e], acc[e]);
    }
    m = to;
  }
  if ((int)r0 + lane / LPR >= rows) return;
  const uint32_t row = block * ROWS + r, G = p.group;
  const int i = row / G, h = hk * G + row % G;
  const bool empty = !(l > 0.0f);  // zero or NaN
  const float inv = empty ? 1.0f : 1.0f / l;
  char* dst = (char*)p.o + 2 * ((long long)(sp.sq.q0 + i) * p.o_st + (long long)h * p.o_sh + lane % LPR * 4);
  *(u32x2*)dst = (u32x2){pack2(acc[0] * inv, acc[1] * inv, F16), pack2(acc[2] * inv, acc[3] * inv, F16)};
  if (lane % LPR == 0)
    p.lse[(long long)h * p.lse_h + (long long)(sp.sq.q0 + i) * p.lse_t] =
        empty ? __builtin_huge_valf() : (m + __log2f(l)) * 0.69314718055994530942f;
}

}  // namespace g950

extern "C" __global__ __launch_bounds__(64) void g950_attn_tree_general(const g950::AttnTreeArgs p) {
  g950::attn_tree_general_body(p);
}
#define G950_TREE_MERGE(NAME, D, F16, RW, NW)                                                               \
  extern "C" __global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void NAME(const g950::AttnTreeArgs p) { \
    g950::attn_tree_merge_body<D, F16, 32 * RW, NW>(p);                                                     \
  }
#define G950_TREE(NAME, D, F16, RW, PER_CU)                                                                 \
  extern "C" __global__ __launch_bounds__(256, PER_CU) void NAME##_r##RW(const g950::AttnTreeArgs p) {      \
    g950::attn_tree_body<D, F16, RW>(p);                                                                    \
  }                                                                                                         \
  G950_TREE_MERGE(NAME##_r##RW##_merge1, D, F16, RW, 1)                                                      \
  G950_TREE_MERGE(NAME##_r##RW##_merge4, D, F16, RW, 4)                                                      \
  G950_TREE_MERGE(NAME##_r##RW##_merge16, D, F16, RW, 16)
#define G950_TREE_SET(TNAME, F16)                          \
  G950_TREE(g950_attn_tree_##TNAME##_d64, 64, F16, 2, 2)   \
  G950_TREE(g950_attn_tree_##TNAME##_d64, 64, F16, 4, 2)   \
  G950_TREE(g950_attn_tree_##TNAME##_d128, 128, F16, 2, 2) \
  G950_TREE(g950_attn_tree_##TNAME##_d128, 128, F16, 4, 2) \
  G950_TREE(g950_attn_tree_##TNAME##_d256, 256, F16, 2, 1) \
  G950_TREE(g950_attn_tree_##TNAME##_d256, 256, F16, 4, 1)
G950_TREE_SET(bf16, false)
G950_TREE_SET(f16, true)
