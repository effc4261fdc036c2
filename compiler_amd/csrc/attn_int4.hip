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
// Lanes take keys for the scores, dims for O.  A cache row is read once for every
// query row and head, 64 rows apart: bound by the latency of its loads.
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

// ---------------------------------------------------------------- fast form
// d 64, 128 or 256, pages of whole 16-key runs, 16-byte rows.  A workgroup owns
// one (sequence, KV head, block of 16 RT query rows, key range); a query row is
// (query, head of the group), so K and V are read once for the whole group.  Its
// 4 or 16 waves take 32-key tiles in turn and share nothing until the end: each fills
// its own LDS ring by direct global->LDS DMA and waits for its own loads only.
//
// What bounds it is the vector ALU beside the bytes: a tile of 32 keys is 64 d values in
// 64 lanes; its 4.4 KB (d 128) come from HBM in 0.75 us where all 1024 SIMDs load, and a
// SIMD with four waves works on it for 0.63 us.  No value is therefore ever dequantised:
// the matrix cores multiply the codes, and scale and offset enter where a tile has few
// numbers.
//   * A word holds 8 codes; (w >> 4 i) & 0x000F000F | bias makes two of them
//     numbers at once, 128 + c in bfloat16 or 64 + c in float16 (the code lands in the
//     mantissa): 7 operations for 8 codes.
//   * S = s (sum q c) + o sum q, c in -8 .. 7: the bias leaves through the MFMA's
//     addend, -(bias + 8) sum q.  Exact products, fp32 sums.
//   * O = sum (p s) c + sum p o: the probability carries V's scale, rounded to
//     bfloat16 once, or to two bfloat16 terms in float16 models (its range, as s may be
//     any size); the bias leaves through one
//     more MFMA with a constant -136 in place of V, over the same rounded values, so
//     that nothing of it is left.  p o and the softmax sum stay in fp32.
//   * V^T needs keys along the contraction: a lane reads the same word of its four
//     keys of each half, and byte permutes put two keys beside each other before
//     the masks; no transpose.  Lane (g, l)'s keys are g + 4 e of each half, so the
//     four rows of a read lie in different LDS banks.
//   * K's dims are taken in the order in which the words hold them; q's fragments
//     are laid out to match, once.
// Measured, in us (32 query heads on 8 KV heads, d 128, bfloat16, pages of 64), in runs of 23
// launches after a pause; in a run of thousands what the vector ALU bounds takes a tenth less
// (the 32 sequences 23.8, the chunks 108.6, 426 TFLOP/s), the rest as long:
//   64 sequences of 8192 keys  114, 5.0 TB/s (a plain copy: 6.0)
//   3 of 65537 to 81920        51.7 and 5.2 for joining the parts, 4.7 TB/s
//   32 of 300 to 4096          25.5 (77 MB; the longest sequences' workgroups end last)
//   1 of 1000                  11.5: 6.2 with a single key, then 0.6 per tile of a SIMD
//   2 of 301 to 512 queries behind 3001 to 4096 keys: 120, 386 TFLOP/s; a tile's codes are
//     unpacked again for every 32 query rows, and 72% of the CUs' time is used (800
//     workgroups on 512 places)
// 16 sequences of 4 queries, 8 heads on one KV head, d 64, float16, 511 to 8192 keys: 11.4
// and 3.9.
constexpr int I4_TK = 32;  // keys per tile of one wave

__device__ __forceinline__ void dma_lane16(const char* src, uint32_t lds_dst) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds_dst);
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}
// the same from a wave-uniform base and a 32-bit lane offset
__device__ __forceinline__ void dma_base16(const char* base, uint32_t off, uint32_t lds_dst) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds_dst);
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(m0) : "memory");
}
__device__ __forceinline__ void dma_lane4(const char* src, uint32_t lds_dst) {
  const uint32_t m0 = __builtin_amdgcn_readfirstlane(lds_dst);
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "{m0}"(m0) : "memory");
}

template <bool F16>
__device__ __forceinline__ f32x4 int4_mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// scale (low half) and offset (high half) of a pair
template <bool F16>
__device__ __forceinline__ void int4_pair(uint32_t w, float& s, float& o) {
  if constexpr (F16) {
    s = f16_to_f32((uint16_t)w);
    o = f16_to_f32((uint16_t)(w >> 16));
  } else {
    s = __uint_as_float(w << 16);
    o = __uint_as_float(w & 0xFFFF0000u);
  }
}

// Two codes of a word as numbers, (shifted word & mask) | bias, in one operation beside
// the shift: with both constants as literals the compiler takes two, so they are
// kept in registers that it cannot see through.  (Not the instruction itself in inline
// asm: the wait states that an MFMA needs behind the writer of its operand are not
// inserted behind asm.)  bfloat16: the code in mantissa bits 0 .. 3 of 128; float16: bits
// 4 .. 7 of 64 (bits 0 .. 3 of 1024 would cost the scores three more bits).
template <bool F16>
struct Int4Codes {
  static constexpr float KOFF = F16 ? 72.0f : 136.0f;  // bias + 8 of K's codes
  uint32_t kmask = F16 ? 0x00F000F0u : 0x000F000Fu, kbias = F16 ? 0x54005400u : 0x43004300u;
  uint32_t vmask = 0x000F000Fu, vbias = 0x43004300u;
  __device__ __forceinline__ Int4Codes() { asm("" : "+s"(kmask), "+v"(kbias), "+s"(vmask), "+v"(vbias)); }
  // codes r and r + 4
  __device__ __forceinline__ uint32_t k(uint32_t w, int r) const {
    if constexpr (F16) w = r == 0 ? w << 4 : w >> (4 * (r - 1));
    else w >>= 4 * r;
    return (w & kmask) | kbias;
  }
  __device__ __forceinline__ uint32_t v(uint32_t w, int r) const { return ((w >> (4 * r)) & vmask) | vbias; }
};

// 8 dims of a query row as pairs (r, r + 4), the order in which a word's codes are
// taken; their sum is added to s
template <bool F16>
__device__ __forceinline__ u32x4 int4_query(const char* src, float& s) {
  const u32x4 w = *(const u32x4*)src;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float a, b;
    int4_pair<F16>(w[e], a, b);
    s += a + b;
  }
  return (u32x4){__builtin_amdgcn_perm(w[2], w[0], 0x05040100u), __builtin_amdgcn_perm(w[2], w[0], 0x07060302u),
                 __builtin_amdgcn_perm(w[3], w[1], 0x05040100u), __builtin_amdgcn_perm(w[3], w[1], 0x07060302u)};
}

// value of `v` combined over the four lanes holding one query row
template <class Op>
__device__ __forceinline__ float int4_row(float v) {
  v = Op::apply(v, __shfl_xor(v, 16));
  return Op::apply(v, __shfl_xor(v, 32));
}

// the largest of three (fmaxf quiets each of its operands first: an operation more each)
__device__ __forceinline__ float int4_max3(float a, float b, float c) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}

// Keys of a sequence that its queries (those the grid covers) see, in tiles of 64:
// from kbeg on, n of them; n = 0 where there is no query, else at least 1.
struct Int4Span {
  Int4Seq sq;
  int nq, nk;       // queries covered, keys that can be read
  long long base;   // visible keys of query i: [base + i - left, base + i + right]
  int kbeg, n;
  __device__ __forceinline__ int first_key(const AttnInt4Args& p, int i) const {
    const long long k = base + i - p.left;
    return p.left < 0 || k < 0 ? 0 : k > nk ? nk : (int)k;
  }
  __device__ __forceinline__ int last_key(const AttnInt4Args& p, int i) const {
    const long long k = base + i + p.right;
    return p.right < 0 || k >= nk ? nk - 1 : k < -1 ? -1 : (int)k;
  }
};
__device__ __forceinline__ Int4Span int4_span(const AttnInt4Args& p, int z) {
  Int4Span s;
  s.sq = int4_seq(p, z);
  s.nq = min(s.sq.nq, p.seqlen_q);
  s.nk = p.pages > 0 ? s.sq.nk : 0;
  s.base = (long long)p.used[z] - s.sq.nq;
  s.kbeg = s.first_key(p, 0) / 64 * 64;
  s.n = s.nq > 0 ? max(1, (s.last_key(p, s.nq - 1) + 1 - s.kbeg + 63) / 64) : 0;
  return s;
}

// What a workgroup does: tiles t0 .. t1 - 1 of a block of query rows of a
// (sequence, KV head); rec: where its partial rows go, -1 if it has all the tiles.
// A sequence's tiles are cut into at most `splits` parts of at least 4 by its own
// length, which lives on the device: short sequences leave no part far longer than
// others'.  Workgroups that share a CU are about a multiple of 256 apart: the
// sequence moves on with the part, so that they differ in length where the batch does.
struct Int4Part {
  int z, hk, block, t0, t1, rec;
};
// tiles of a part, of n
__device__ __forceinline__ int int4_part(const AttnInt4Args& p, int n) {
  return max((int)((uint32_t)(n + p.splits - 1) / (uint32_t)p.splits), 4);
}
__device__ __forceinline__ Int4Part int4_deal(const AttnInt4Args& p, Int4Span& sp) {
  // (unsigned: a division is a third shorter)
  const uint32_t heads = p.Hkv, pairs = p.B * heads, units = pairs * p.row_blocks;
  const uint32_t split = blockIdx.x / units, unit = blockIdx.x % units, pair = unit % pairs;
  Int4Part w;
  w.z = (pair / heads + split * (uint32_t)p.turn) % (uint32_t)p.B;
  w.hk = pair % heads;
  w.block = p.row_blocks - 1 - (int)(unit / pairs);  // those that see most keys first
  sp = int4_span(p, w.z);
  const int c = int4_part(p, sp.n);
  w.t0 = (int)split * c;
  w.t1 = min(sp.n, w.t0 + c);
  w.rec = sp.n <= c ? -1 : ((w.z * p.Hkv + w.hk) * p.row_blocks + w.block) * p.splits + split;
  return w;
}

// The waves' partial rows of a workgroup joined: row r's O unnormalised in wave w's
// LDS (16-byte chunks XOR-swizzled by the row), its maximum (log2 units) and sum in
// ml[w][r].  Writes o and lse, or record rec0.
template <int D, bool F16, int ROWS, int WLDS, int NW>
__device__ __forceinline__ void int4_finish(const AttnInt4Args& p, const char* lds, const float* ml, const Int4Seq& sq,
                                            int hk, int rec0, int row0, int nrows) {
  const uint32_t G = p.group;
  constexpr int CPR = D / 4;  // 16-byte chunks (4 d) per row
  for (int it = threadIdx.x; it < nrows * CPR; it += NW * 64) {
    const int r = it / CPR, c = it % CPR;
    float m = ml[2 * r];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, ml[2 * (w * ROWS + r)]);
    f32x4 sum = {};
    float lt = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float mw = ml[2 * (w * ROWS + r)], lw = ml[2 * (w * ROWS + r) + 1];
      // no finite score: no key of this row (l = 0), or only NaN ones
      const float f = mw == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
      lt = fmaf(f, lw, lt);
      const f32x4 ow = *(const f32x4*)(lds + w * WLDS + r * D * 4 + ((c ^ (r & 15)) << 4));
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, ow[e], sum[e]);
    }
    if (rec0 >= 0) {
      const long long rec = (long long)rec0 * ROWS + r;
      *(f32x4*)(p.part + rec * D + c * 4) = sum;
      if (c == 0) {
        p.ml[2 * rec] = m;
        p.ml[2 * rec + 1] = lt;
      }
      continue;
    }
    const int i = (uint32_t)(row0 + r) / G, h = hk * G + (uint32_t)(row0 + r) % G;
    const bool empty = !(lt > 0.0f);  // zero or NaN
    const float inv = empty ? 1.0f : 1.0f / lt;
    char* dst = (char*)p.o + 2 * ((long long)(sq.q0 + i) * p.o_st + (long long)h * p.o_sh + c * 4);
    if constexpr (F16)
      *(u32x2*)dst = (u32x2){__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){sum[0] * inv, sum[1] * inv}, f16x2)),
                             __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){sum[2] * inv, sum[3] * inv}, f16x2))};
    else
      *(u32x2*)dst = (u32x2){__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){sum[0] * inv, sum[1] * inv}, bf16x2)),
                             __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){sum[2] * inv, sum[3] * inv}, bf16x2))};
    if (c == 0)
      p.lse[(long long)h * p.lse_h + (long long)(sq.q0 + i) * p.lse_t] =
          empty ? __builtin_huge_valf() : (m + __log2f(lt)) * 0.69314718055994530942f;
  }
}

template <int D, bool F16, int RT, int NW>
__device__ __forceinline__ void attn_int4_body(const AttnInt4Args& p) {
  constexpr int RB = D / 2;                       // bytes of a row
  constexpr int KT = I4_TK * RB;                  // bytes of a tile's K (or V)
  constexpr int TILE = 2 * KT + 256;              // K, V, 64 pairs
  constexpr int PAIRS = 512;                      // the pairs of one tile in fp32
  // tiles in flight per wave: four workgroups share a CU's 160 KiB with one row tile (36 and
  // 38 KiB at d 128 and 64), three with two at d 64 (48), two at d 128 and with d 256 (69 and
  // 70), one of 16 waves
  constexpr int ST = RT == 1 ? (D == 64 ? 4 : 2) : (D == 64 ? 5 : 4);
  constexpr int RING = ST * TILE + PAIRS;
  constexpr int DC = KT / 1024;                   // DMA instructions of a tile's K
  constexpr int DPT = 2 * DC + 1;
  constexpr int LPK = RB / 16;                    // lanes (16 bytes) per key of a DMA instruction
  constexpr int KPI = 64 / LPK;                   // keys per instruction
  constexpr int KS = D / 32;                      // words of a lane per K row: k-steps of S^T
  constexpr int VW = D == 256 ? 2 : 1;            // words (d 64: half words) of a lane per V row
  constexpr int VN = D == 64 ? 4 : 8;             // codes of each
  constexpr int NB = VW * VN;                     // 16-d blocks of O^T
  constexpr int ROWS = 16 * RT;
  constexpr int PT = F16 ? 2 : 1;                 // bfloat16 terms of a probability
  constexpr int WLDS = RING > ROWS * D * 4 ? RING : ROWS * D * 4;  // a wave's LDS: its ring, then its partial O
  __shared__ __attribute__((aligned(1024))) char lds[NW * WLDS];
  __shared__ float ml[NW][ROWS][2];
  if (blockDim.x != NW * 64) return;  // launch shape must match the kernel
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g4 = lane >> 4, l16 = lane & 15;
  const uint32_t G = p.group;
  Int4Span sp;
  const Int4Part w = int4_deal(p, sp);
  const int hk = w.hk;
  const Int4Seq& sq = sp.sq;
  const int rows = sp.nq * p.group;  // of this sequence and KV head
  const int row0 = w.block * ROWS;
  if (row0 >= rows || w.t0 >= sp.n) return;
  const int nrows = min(ROWS, rows - row0);
  auto first_key = [&](int i) { return sp.first_key(p, i); };
  auto last_key = [&](int i) { return sp.last_key(p, i); };
  const int i_lo = (uint32_t)row0 / G, i_hi = (uint32_t)(row0 + nrows - 1) / G;
  const int all_from = first_key(i_hi), all_to = last_key(i_lo);  // keys every row sees
  const int lo = max(sp.kbeg + 64 * w.t0, first_key(i_lo) / I4_TK * I4_TK);
  const int hi = min(last_key(i_hi) + 1, w.t1 < sp.n ? sp.kbeg + 64 * w.t1 : 0x7FFFFFFF);

  // query fragments: row l16 of tile rt; lane group g4 holds dims g4 D / 4 ..,
  // word ks their 8 from 8 ks on, as pairs (r, r + 4)
  u32x4 qf[RT][KS];
  float qsum[RT];
  int kmin[RT], kmax[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const uint32_t r = row0 + min(rt * 16 + l16, nrows - 1);
    const int i = r / G, h = hk * G + r % G;
    kmin[rt] = first_key(i);
    kmax[rt] = last_key(i);
    const char* src = (const char*)p.q + 2 * ((long long)(sq.q0 + i) * p.q_st + (long long)h * p.q_sh + g4 * (D / 4));
    float s = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[rt][ks] = int4_query<F16>(src + ks * 16, s);
    }
    qsum[rt] = int4_row<OpSum>(s);
  }

  char* ring = lds + wave * WLDS;
  const uint32_t ring32 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)ring;
  const char* kbase = (const char*)p.k + (long long)hk * p.k_h;
  const char* vbase = (const char*)p.v + (long long)hk * p.v_h;
  // this lane's share of a DMA instruction: key dkey (of KPI), 16-byte piece dpos
  const int dkey = lane / LPK, dpos = lane % LPK;
  const uint32_t koff = (dkey & 15) * (uint32_t)p.k_r + dpos * 16, voff = (dkey & 15) * (uint32_t)p.v_r + dpos * 16;
  // and of the pairs: word lane = ((kind * 2 + half) * 4 + g) * 4 + e holds key g + 4 e of the half
  const int skey = ((lane >> 2) & 3) + 4 * (lane & 3), shalf = (lane >> 4) & 1;
  const char* sbase = lane < 32 ? (const char*)p.ks + 2 * ((long long)hk * p.ks_h + (long long)skey * p.ks_r)
                                : (const char*)p.vs + 2 * ((long long)hk * p.vs_h + (long long)skey * p.vs_r);
  const uint32_t s_p = 2 * (uint32_t)(lane < 32 ? p.ks_p : p.vs_p), s_r = 2 * (uint32_t)(lane < 32 ? p.ks_r : p.vs_r);
  const int* table = p.table + (long long)w.z * p.table_s;
  const int ntiles = hi > lo ? (hi - lo + I4_TK - 1) / I4_TK : 0;
  const int nloc = ntiles > wave ? (ntiles - wave + NW - 1) / NW : 0;
  // of this wave's tiles, those whose every key every row sees: free_from .. free_to - 1
  auto own_tiles = [&](int keys) { return keys < 0 ? 0 : (keys / I4_TK - wave + NW - 1) / NW; };
  const int free_from = own_tiles(all_from - lo + I4_TK - 1), free_to = own_tiles(min(all_to + 1, hi) - lo);

  // pages and rows of this wave's next 32 tiles, one 16-key half per lane; a half
  // without a page (or past the end) reads page 0 and is masked
  int pages = 0, prow = 0;
  uint64_t live[2] = {0, 0};  // by the parity of the batch of 32 tiles
  auto issue = [&](int j) {
    if ((j & 31) == 0) {
      const int key = lo + I4_TK * (wave + NW * (j + (lane >> 1))) + 16 * (lane & 1);
      const int e = key / p.block_size;
      int ph = key < hi && e < p.max_pages ? table[e] : -1;
      ph = ph < p.pages ? ph : -1;
      const uint64_t m = __ballot(ph >= 0);
      if (j & 32) live[1] = m;
      else live[0] = m;
      prow = ph < 0 ? 0 : key - e * p.block_size;
      pages = max(ph, 0);
    }
    const int at = 2 * (j & 31);
    const int pg[2] = {__builtin_amdgcn_readlane(pages, at), __builtin_amdgcn_readlane(pages, at + 1)};
    const int pr[2] = {__builtin_amdgcn_readlane(prow, at), __builtin_amdgcn_readlane(prow, at + 1)};
    const uint32_t dst = ring32 + (j % ST) * TILE;
    const char *ksrc[2], *vsrc[2];
    // (unsigned halves: a 64-bit product of them is three scalar multiplies, or two)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      ksrc[t] = kbase + (uint32_t)pg[t] * (uint64_t)p.k_p + (uint64_t)(uint32_t)pr[t] * (uint32_t)p.k_r;
      vsrc[t] = vbase + (uint32_t)pg[t] * (uint64_t)p.v_p + (uint64_t)(uint32_t)pr[t] * (uint32_t)p.v_r;
    }
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
      for (int u = 0; u < DC; ++u) {
        const char* const* src = kind ? vsrc : ksrc;
        const uint32_t to = dst + (kind ? KT : 0) + u * 1024, off = kind ? voff : koff;
        if constexpr (KPI <= 16)
          dma_base16(src[u * KPI / 16], off + u * KPI % 16 * (uint32_t)(kind ? p.v_r : p.k_r), to);
        else
          dma_lane16((dkey < 16 ? src[0] : src[1]) + off, to);
      }
    const uint32_t pl = shalf ? pg[1] : pg[0], rl = shalf ? pr[1] : pr[0];
    dma_lane4(sbase + (uint64_t)pl * s_p + (uint64_t)rl * s_r, dst + 2 * KT);
  };

  f32x4 o[RT][NB], ob[RT];
  float ms[RT], l[RT], zo[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    ms[rt] = -__builtin_huge_valf();
    l[rt] = zo[rt] = 0.0f;
    ob[rt] = (f32x4){};
#pragma unroll
    for (int b = 0; b < NB; ++b) o[rt][b] = (f32x4){};
  }
  const float unit = lane < 32 ? p.scale_log2 : 1.0f;
  const char* const pairs = ring + ST * TILE + 32 * g4;
  const Int4Codes<F16> two;
  const int kperm = (l16 >> 2) + 4 * (l16 & 3);  // K row of S^T's row l16
  const uint32_t m136 = 0xC308C308u;             // -136 in bfloat16, twice
  const u32x4 unbias = {m136, m136, m136, m136};
  for (int j = 0; j < ST && j < nloc; ++j) issue(j);
  for (int i = 0; i < nloc; ++i) {
    // tile i has landed once at most the later tiles' loads are in flight
    if (i + ST <= nloc) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((ST - 1) * DPT) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const char* st = ring + (i % ST) * TILE;
    const int kv0 = lo + I4_TK * (wave + NW * i);
    // every lane decodes one of the 64 pairs (K's in log2 units) for all of them: read
    // back once K is unpacked
    {
      float sc, of;
      int4_pair<F16>(*(const uint32_t*)(st + 2 * KT + 4 * lane), sc, of);
      *(f32x2*)(ring + ST * TILE + 8 * lane) = (f32x2){sc * unit, of * unit};
    }
    f32x4 s[2][RT];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t kw[KS];
      const char* kr = st + (t * 16 + kperm) * RB + g4 * (RB / 4);
      if constexpr (KS == 2) {
        const u32x2 w = *(const u32x2*)kr;
        kw[0] = w[0];
        kw[1] = w[1];
      } else {
#pragma unroll
        for (int c = 0; c < KS / 4; ++c) {
          const u32x4 w = *(const u32x4*)(kr + 16 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) kw[4 * c + e] = w[e];
        }
      }
      f32x4 acc[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float q = -Int4Codes<F16>::KOFF * qsum[rt];
        acc[rt] = (f32x4){q, q, q, q};
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4 kf;
#pragma unroll
        for (int r = 0; r < 4; ++r) kf[r] = two.k(kw[ks], r);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt] = int4_mfma<F16>(kf, qf[rt][ks], acc[rt]);
      }
      const f32x4 kp[2] = {*(const f32x4*)(pairs + t * 128), *(const f32x4*)(pairs + t * 128 + 16)};
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          s[t][rt][e] = fmaf(kp[e / 2][2 * (e & 1)], acc[rt][e], kp[e / 2][2 * (e & 1) + 1] * qsum[rt]);
    }
    const uint32_t alive = (uint32_t)(live[(i >> 5) & 1] >> (2 * (i & 31))) & 3;
    const bool mask = alive != 3 || i < free_from || i >= free_to;
    if (mask) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = kv0 + 16 * t + g4 + 4 * e;
            if (!((alive >> t) & 1) || key < kmin[rt] || key > kmax[rt] || key >= hi) s[t][rt][e] = -__builtin_huge_valf();
          }
    }
    u32x4 pf[RT][PT];
    float vs[2][4], vo[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const f32x4 vp[2] = {*(const f32x4*)(pairs + 256 + t * 128), *(const f32x4*)(pairs + 256 + t * 128 + 16)};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        vs[t][e] = vp[e / 2][2 * (e & 1)];
        vo[t][e] = vp[e / 2][2 * (e & 1) + 1];
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const float mh = int4_max3(int4_max3(s[0][rt][0], s[0][rt][1], s[0][rt][2]),
                                 int4_max3(s[0][rt][3], s[1][rt][0], s[1][rt][1]),
                                 int4_max3(s[1][rt][2], s[1][rt][3], s[1][rt][3]));
      if (__any(mh > ms[rt] + 8.0f)) {
        const float mt = int4_row<OpMax>(mh);
        const bool move = mt > ms[rt] + 8.0f;
        const float alpha = move ? __builtin_amdgcn_exp2f(ms[rt] - mt) : 1.0f;
        l[rt] *= alpha;
        zo[rt] *= alpha;
        ob[rt] *= alpha;
#pragma unroll
        for (int b = 0; b < NB; ++b) o[rt][b] *= alpha;
        ms[rt] = move ? mt : ms[rt];
      }
      // rows without a visible key so far: exponent base 0, exp2(-inf) = 0
      const float mb = (ms[rt] == -__builtin_huge_valf()) ? 0.0f : ms[rt];
      float ps[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float pe[4], zp[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pe[e] = __builtin_amdgcn_exp2f(s[t][rt][e] - mb);
          ps[t][e] = pe[e] * vs[t][e];
          zp[e] = vo[t][e];
        }
        if (mask) {  // what a row does not see may hold anything
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool none = s[t][rt][e] == -__builtin_huge_valf();
            ps[t][e] = none ? 0.0f : ps[t][e];
            zp[e] = none ? 0.0f : zp[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) zo[rt] = fmaf(pe[e], zp[e], zo[rt]);
        l[rt] += (pe[0] + pe[1]) + (pe[2] + pe[3]);
      }
      // bfloat16 models: one rounding; float16 models: what the rounding left out as a
      // second term (their outputs hold more bits than one term gives them)
#pragma unroll
      for (int n = 0; n < PT; ++n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float* two_p = &ps[j / 2][2 * (j & 1)];
          const uint32_t pk = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){two_p[0], two_p[1]}, bf16x2));
          pf[rt][n][j] = pk;
          if (n + 1 < PT) {
            two_p[0] -= __uint_as_float(pk << 16);
            two_p[1] -= __uint_as_float(pk & 0xFFFF0000u);
          }
        }
        ob[rt] = int4_mfma<false>(unbias, pf[rt][n], ob[rt]);
      }
    }
    // V: words of keys g4 + 4 e of both halves, two keys side by side
    const char* vr = st + KT + g4 * RB + l16 * (D == 64 ? 2 : 4);
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      u32x4 half[D == 64 ? 1 : 2];  // codes 0 .. 3 (and 4 .. 7) of the pairs of keys
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const char* a = vr + (16 * t + 4 * e) * RB + c * 64;
          if constexpr (D == 64) {
            half[0][2 * t + e / 2] = (uint32_t)*(const uint16_t*)a | (uint32_t)*(const uint16_t*)(a + 4 * RB) << 16;
          } else {
            const uint32_t w0 = *(const uint32_t*)a, w1 = *(const uint32_t*)(a + 4 * RB);
            half[0][2 * t + e / 2] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
            half[1][2 * t + e / 2] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
          }
        }
#pragma unroll
      for (int n = 0; n < VN; ++n) {
        u32x4 vf;
#pragma unroll
        for (int r = 0; r < 4; ++r) vf[r] = two.v(half[n / 4][r], n & 3);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int m = 0; m < PT; ++m) o[rt][c * VN + n] = int4_mfma<false>(vf, pf[rt][m], o[rt][c * VN + n]);
      }
    }
    // this tile's LDS reads have returned before its slot is refilled
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (i + ST < nloc) issue(i + ST);
  }

  // ---- the waves' partial rows: O through each wave's own ring (16-byte
  // chunks XOR-swizzled by the row), maxima and sums beside it.  Block b = c VN + n,
  // element e: dim 128 c + VN (4 g4 + e) + n.
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rt * 16 + l16;
    const float ls = int4_row<OpSum>(l[rt]), add = int4_row<OpSum>(zo[rt]) + ob[rt][0];
#pragma unroll
    for (int c = 0; c < VW; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < VN; n += 4) {
          const int chunk = (128 * c + VN * (4 * g4 + e) + n) / 4;
          *(f32x4*)(ring + r * D * 4 + ((chunk ^ l16) << 4)) =
              (f32x4){o[rt][c * VN + n][e] + add, o[rt][c * VN + n + 1][e] + add, o[rt][c * VN + n + 2][e] + add,
                      o[rt][c * VN + n + 3][e] + add};
        }
    if (g4 == 0) {
      ml[wave][r][0] = ms[rt];
      ml[wave][r][1] = ls;
    }
  }
  __syncthreads();
  int4_finish<D, F16, ROWS, WLDS, NW>(p, lds, &ml[0][0][0], sq, hk, w.rec, row0, nrows);
}

// Joins the parts of a block of query rows: one wave per row, lane s holds part s's
// maximum and sum (at most 64 parts), D / 64 outputs per lane.  Latency is all of it, so
// the records are read before the lengths say how many of them there are (what lies
// behind the last one is read and left), 32 loads at a time: 42 parts of 96 rows 5.3 us,
// 6.1 with 8 at a time behind the lengths; 32 parts of 512 rows of 64 dims 3.9 and 4.5.
template <int D, bool F16, int ROWS>
__device__ __forceinline__ void attn_int4_merge_body(const AttnInt4Args& p) {
  const int lane = threadIdx.x & 63;
  // (parts are wanted for a few blocks per CU only: 32 bits hold their rows)
  const uint32_t item = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t id = item / (uint32_t)p.merge_rows, r = item % (uint32_t)p.merge_rows;
  if (id >= (uint32_t)(p.B * p.Hkv * p.row_blocks)) return;
  const uint32_t blocks = p.row_blocks, heads = p.Hkv, pair = id / blocks;
  const int block = id % blocks, z = pair / heads, hk = pair % heads;
  const int row = block * ROWS + r;
  constexpr int E = D / 64, U = 32 / E;
  using vec = float __attribute__((ext_vector_type(E)));
  const long long rec = (long long)id * p.splits * ROWS + r;
  const float* part = p.part + rec * D + lane * E;
  const float* pair_ml = p.ml + 2 * (rec + (long long)min(lane, p.splits - 1) * ROWS);
  float m = pair_ml[0], l = pair_ml[1];
  vec v[U];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = *(const vec*)(part + (long long)min(s0 + u, p.splits - 1) * ROWS * D);
  };
  load(0);
  const Int4Span sp = int4_span(p, z);
  if (row >= sp.nq * p.group) return;
  const int c = int4_part(p, sp.n), count = (sp.n + c - 1) / c;
  if (count <= 1) return;  // its workgroup had all of it
  if (lane >= count) {
    m = -__builtin_huge_valf();
    l = 0.0f;
  }
  const float mt = wave_reduce<OpMax>(m);
  // no finite score in a part: nothing seen (O = l = 0), or only NaN, which stays
  const float f = m == -__builtin_huge_valf() ? 1.0f : __builtin_amdgcn_exp2f(m - mt);
  const float lt = wave_reduce<OpSum>(f * l);
  vec acc = {};
  for (int s0 = 0;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(s0 + u, 63)));
      if (s0 + u < count)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w, v[u][e], acc[e]);
    }
    if ((s0 += U) >= count) break;
    load(s0);
  }
  const int i = (uint32_t)row / (uint32_t)p.group, h = hk * p.group + (uint32_t)row % (uint32_t)p.group;
  const bool empty = !(lt > 0.0f);  // zero or NaN
  const float inv = empty ? 1.0f : 1.0f / lt;
  uint16_t* dst = (uint16_t*)p.o + (long long)(sp.sq.q0 + i) * p.o_st + (long long)h * p.o_sh + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) dst[e] = F16 ? f32_to_f16(acc[e] * inv) : f32_to_bf16(acc[e] * inv);
  if (lane == 0)
    p.lse[(long long)h * p.lse_h + (long long)(sp.sq.q0 + i) * p.lse_t] =
        empty ? __builtin_huge_valf() : (mt + __log2f(lt)) * 0.69314718055994530942f;
}

}  // namespace g950

extern "C" __global__ __launch_bounds__(64) void g950_attn_int4_general(const g950::AttnInt4Args p) {
  g950::attn_int4_general_body(p);
}
// Four workgroups per CU with one row tile (128 registers), three with two at d 64 (two
// chunks of 301 to 512 queries behind 3001 to 4096 keys: 89 us, 98 with two and seven tiles
// in flight), else two (at d 128 a third would spill: 206 us against 119).
#define G950_INT4(NAME, D, F16, RT)                                                                    \
  extern "C" __global__ __launch_bounds__(256, RT == 1 && D < 256 ? 4 : D == 64 ? 3 : 2) void           \
      NAME##_r##RT(const g950::AttnInt4Args p) {                                                       \
    g950::attn_int4_body<D, F16, RT, 4>(p);                                                            \
  }                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void NAME##_r##RT##_merge(const g950::AttnInt4Args p) { \
    g950::attn_int4_merge_body<D, F16, 16 * RT>(p);                                                    \
  }
G950_INT4(g950_attn_int4_bf16_d64, 64, false, 1)
G950_INT4(g950_attn_int4_bf16_d64, 64, false, 2)
G950_INT4(g950_attn_int4_bf16_d128, 128, false, 1)
G950_INT4(g950_attn_int4_bf16_d128, 128, false, 2)
G950_INT4(g950_attn_int4_bf16_d256, 256, false, 1)
G950_INT4(g950_attn_int4_f16_d64, 64, true, 1)
G950_INT4(g950_attn_int4_f16_d64, 64, true, 2)
G950_INT4(g950_attn_int4_f16_d128, 128, true, 1)
G950_INT4(g950_attn_int4_f16_d128, 128, true, 2)
G950_INT4(g950_attn_int4_f16_d256, 256, true, 1)
// 16 waves to a block (one workgroup per CU): where a CU has a block or two of some
// length, and parts would only be joined again.
#define G950_INT4W(NAME, D, F16)                                                                   \
  extern "C" __global__ __launch_bounds__(1024) void NAME##_r1w(const g950::AttnInt4Args p) {     \
    g950::attn_int4_body<D, F16, 1, 16>(p);                                                        \
  }
G950_INT4W(g950_attn_int4_bf16_d64, 64, false)
G950_INT4W(g950_attn_int4_bf16_d128, 128, false)
G950_INT4W(g950_attn_int4_f16_d64, 64, true)
G950_INT4W(g950_attn_int4_f16_d128, 128, true)
