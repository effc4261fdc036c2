// Appending keys and values to a paged cache on gfx950, with the position
// rotation of queries and keys on the way.  Token t of sequence b (rows
// cu[b] .. cu[b + 1] - 1) stands at position
//   p = used[b] - (cu[b + 1] - cu[b]) + t - cu[b]
// (used counts the new keys too), and goes to row p % block_size of page
// table[b, p / block_size].  The first R dims of q and k turn in pairs, (i, i +
// R / 2) or (2i, 2i + 1), by row p of the cos / sin tables:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// in fp32, rounded once.  The two products and their sum round separately (no
// fused multiply-add), so that a 4-bit code does not depend on how the compiler
// contracts them.
//
// 4-bit rows: a (token, head) row x of D dims, after the rotation and before
// any rounding, is held as
//   s = T((max - min) / 15), o = T(min + 8 s), c = clamp(rint((x - o) (1 / s)) + 8, 0, 15)
// and stands for (c - 8) s + o; T is the model's type.  Byte i holds dims 2i
// (low half) and 2i + 1.  A row whose spread rounds to nothing has s = 0 and o = its
// value; a row that holds NaN or infinities (or whose spread passes fp32) has s = o = NaN.
// s and o round once, as they are kept, and the codes are taken against the rounded pair, so
// that its rounding moves the codes and the values stay within half a step s; but at the row's
// ends the codes clamp, and a value is off by up to o's rounding and 15 of s's (2^-8 of each
// in bfloat16, 2^-11 in float16) where that is more: rows far from 0 beside their
// spread lose one end.
//
// Trees of drafted tokens (TREE): node i of a sequence has a parent among the nodes before
// it, or none (any other value); it goes to the cache row of position used - n + i, n the
// sequence's nodes, and stands at position used - n + depth, where the rotation is concerned.
// The depth is a walk in registers over parents loaded 64 at a time, beside the loads of the
// rows: 3.4 thousand nodes of 64 trees (32 + 8 + 8 heads of 128 in bfloat16, 83 MB) 18 us, 4.6 TB/s.
// The walk is as long as a node is deep: a chain of 256 nodes 17 us, of 1024 82 (the plain append, which does the same
// to a chain, 7); trees of that many nodes two levels deep 7 and 8.
//
// Nothing is written for tokens past cu[B] or of a sequence whose rows are not
// rows of q; nor, at a position below 0 or past the tables; a page that the
// table or the pool does not hold drops only the cache row.
#include <type_traits>

namespace g950 {

// Where a token goes (the same for all lanes of a wave).
struct KvPlace {
  int seq, pos;       // seq < 0: nothing to do
  int page;           // < 0: no cache row
  int row;
};

// The sequence of token t: the last one that starts at or before it, found by
// 64 starts at a time, checked to hold it.
__device__ __forceinline__ int kv_sequence(const int* cu, int B, int T, int t, int& b0, int& b1) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B + 1;
  while (n > 64) {
    const int step = (n + 63) >> 6;
    const int i = lane * step;
    const int c = __popcll(__ballot(i < n && cu[lo + (i < n ? i : 0)] <= t));
    if (c == 0) return -1;
    const int skip = (c - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  const int c = __popcll(__ballot(lane < n && cu[lo + (lane < n ? lane : 0)] <= t));
  const int b = lo + c - 1;
  if (c == 0 || b >= B) return -1;
  b0 = cu[b];
  b1 = cu[b + 1];
  return b0 >= 0 && t >= b0 && t < b1 && b1 <= T ? b : -1;
}

// Levels above node i of the tree whose parents begin at `parent`: the way to its root
// through 64 parents at a time, one per lane (a node's parent lies below it; all
// arguments are wave-uniform).
__device__ __forceinline__ int kv_depth(const int* parent, int i) {
  const int lane = threadIdx.x & 63;
  int depth = 0, from = i + 1, up = 0;
  for (;;) {
    if (i < from) {
      from = max(i - 63, 0);
      up = parent[min(from + lane, i)];
    }
    const int p = __builtin_amdgcn_readlane(up, i - from);
    if (p < 0 || p >= i) return depth;
    ++depth;
    i = p;
  }
}

template <bool TREE>
__device__ __forceinline__ KvPlace kv_place(const KvAppendArgs& a, int t) {
  KvPlace w;
  w.pos = w.row = 0;
  w.page = -1;
  int b0 = 0, b1 = 0;
  w.seq = __builtin_amdgcn_readfirstlane(kv_sequence(a.cu, a.B, a.T, t, b0, b1));
  if (w.seq < 0) return w;
  long long pos = (long long)a.used[w.seq] - (b1 - b0) + (t - b0);
  const int slot = __builtin_amdgcn_readfirstlane((int)pos);
  if constexpr (TREE) {
    b0 = __builtin_amdgcn_readfirstlane(b0);
    pos += kv_depth(a.parent + b0, t - b0) - (t - b0);
  }
  if (pos < 0 || (a.R && pos >= a.positions)) {
    w.seq = -1;
    return w;
  }
  w.pos = __builtin_amdgcn_readfirstlane((int)pos);
  const int e = slot / a.block_size;
  w.row = slot % a.block_size;
  if (e < a.max_pages) {
    const int ph = a.table[(long long)w.seq * a.table_s + e];
    w.page = ph >= 0 && ph < a.pages ? ph : -1;
  }
  w.page = __builtin_amdgcn_readfirstlane(w.page);
  return w;
}

// an fp32 value as it stands: neither a sum draws the product before it into a
// fused multiply-add (-ffp-contract=fast does so whatever a pragma says) nor a
// conversion to float16 the operation before it into one rounding
__device__ __forceinline__ float kv_keep(float v) {
  asm("" : "+v"(v));
  return v;
}

// (a, b) turned; each operation rounds on its own
__device__ __forceinline__ void kv_turn(float a, float b, float c, float s, float& y, float& z) {
  y = kv_keep(a * c) - kv_keep(b * s);
  z = kv_keep(b * c) + kv_keep(a * s);
}

// value rounded to the model's type (dtype code) and back
__device__ __forceinline__ float kv_round(float v, int dt) {
  v = kv_keep(v);
  if (dt == DT_BF16) return bf16_to_f32(f32_to_bf16(v));
  return f16_to_f32(f32_to_f16(v));
}

// A row's scale, offset and reciprocal scale from its least and greatest value.
struct KvScale {
  float s, o, inv;
};
__device__ __forceinline__ KvScale kv_scale(float lo, float hi, bool nan, int dt) {
  KvScale r;
  const float d = hi - lo;
  if (nan || !(d < __builtin_huge_valf())) {
    r.s = r.o = __builtin_nanf("");
    r.inv = 0.0f;
    return r;
  }
  r.s = kv_round(d / 15.0f, dt);
  if (r.s < 0x1p-126f) r.s = 0.0f;
  r.o = kv_round(fmaf(8.0f, r.s, lo), dt);
  r.inv = r.s > 0.0f ? 1.0f / r.s : 0.0f;
  return r;
}
__device__ __forceinline__ int kv_code(float x, const KvScale& k) {
  const float c = rintf((x - k.o) * k.inv) + 8.0f;  // (NaN: 0)
  return (int)fminf(fmaxf(c, 0.0f), 15.0f);
}
__device__ __forceinline__ float kv_value(int c, const KvScale& k) {
  return kv_keep(fmaf((float)(c - 8), k.s, k.o));  // the product is exact
}

// One wave per (token, head) row: any D, R, stride and alignment.  Each row looks its
// place up and each element reads its own cos and sin: 988 us where the vector kernel
// takes 103 (26 thousand tokens, below), 489 against 44 into 4 bits.
template <bool TREE>
__device__ __forceinline__ void kv_append_general_body(const KvAppendArgs& a) {
  const int lane = threadIdx.x & 63;
  const int slots = a.Hq + 2 * a.Hkv;
  const long long tasks = (long long)a.T * slots;
  const int isz = a.dtype == DT_F32 ? 4 : 2;
  for (long long task = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); task < tasks; task += (long long)gridDim.x * 4) {
    const int t = __builtin_amdgcn_readfirstlane((int)(task / slots));
    const int slot = __builtin_amdgcn_readfirstlane((int)(task % slots));
    const KvPlace w = kv_place<TREE>(a, t);
    if (w.seq < 0) continue;
    const bool is_q = slot < a.Hq, is_v = slot >= a.Hq + a.Hkv;
    const int h = is_q ? slot : is_v ? slot - a.Hq - a.Hkv : slot - a.Hq;
    const char* src = is_q ? (const char*)a.q + isz * (t * a.q_st + h * a.q_sh)
                           : is_v ? (const char*)a.v + isz * (t * a.v_st + h * a.v_sh)
                                  : (const char*)a.k + isz * (t * a.k_st + h * a.k_sh);
    const int R = is_v ? 0 : a.R, half = R / 2;
    const long long crow = w.pos * a.cos_s, srow = w.pos * a.sin_s;
    auto at = [&](int d) { return load_as_f32(src, d, a.dtype); };
    auto pair = [&](int i, float& y, float& z) {  // the turned pair i
      const int d0 = a.interleaved ? 2 * i : i, d1 = a.interleaved ? 2 * i + 1 : i + half;
      kv_turn(at(d0), at(d1), load_as_f32(a.cos, crow + i, a.table_dtype), load_as_f32(a.sin, srow + i, a.table_dtype), y,
              z);
    };
    if (is_q || !a.int4) {
      if (!is_q && w.page < 0) continue;
      char* dst = is_q ? (char*)a.q_out + isz * (t * a.qo_st + h * a.qo_sh)
                       : is_v ? (char*)a.v_cache + isz * (w.page * a.vc_p + w.row * a.vc_r + h * a.vc_h)
                              : (char*)a.k_cache + isz * (w.page * a.kc_p + w.row * a.kc_r + h * a.kc_h);
      for (int i = lane; i < half; i += 64) {
        float y, z;
        pair(i, y, z);
        store_from_f32(dst, a.interleaved ? 2 * i : i, a.dtype, y);
        store_from_f32(dst, a.interleaved ? 2 * i + 1 : i + half, a.dtype, z);
      }
      for (int d = R + lane; d < a.D; d += 64) store_from_f32(dst, d, a.dtype, at(d));
      continue;
    }
    auto value = [&](int d) {
      if (d >= R) return at(d);
      float y, z;
      const int i = a.interleaved ? d >> 1 : d < half ? d : d - half;
      pair(i, y, z);
      return (a.interleaved ? (d & 1) == 0 : d < half) ? y : z;
    };
    float lo = __builtin_huge_valf(), hi = -__builtin_huge_valf();
    bool nan = false;
    for (int d = lane; d < a.D; d += 64) {
      const float x = value(d);
      nan |= x != x;
      lo = fminf(lo, x);
      hi = fmaxf(hi, x);
    }
    lo = -wave_reduce<OpMax>(-lo);
    hi = wave_reduce<OpMax>(hi);
    const KvScale k = kv_scale(lo, hi, __any(nan), a.dtype);
    void* out = is_v ? a.v_out : a.k_out;
    const long long oo = is_v ? t * a.vo_st + h * a.vo_sh : t * a.ko_st + h * a.ko_sh;
    uint8_t* dst = is_v ? (uint8_t*)a.v_cache + (w.page * a.vc_p + w.row * a.vc_r + h * a.vc_h)
                        : (uint8_t*)a.k_cache + (w.page * a.kc_p + w.row * a.kc_r + h * a.kc_h);
    for (int i = lane; i < a.D / 2; i += 64) {
      const int c0 = kv_code(value(2 * i), k), c1 = kv_code(value(2 * i + 1), k);
      if (w.page >= 0) dst[i] = (uint8_t)(c0 | c1 << 4);
      if (out) {
        store_from_f32(out, oo + 2 * i, a.dtype, kv_value(c0, k));
        store_from_f32(out, oo + 2 * i + 1, a.dtype, kv_value(c1, k));
      }
    }
    if (lane == 0 && w.page >= 0) {
      void* sc = is_v ? a.v_scale : a.k_scale;
      const long long so = is_v ? w.page * a.vs_p + w.row * a.vs_r + h * a.vs_h
                                : w.page * a.ks_p + w.row * a.ks_r + h * a.ks_h;
      store_from_f32(sc, so, a.dtype, k.s);
      store_from_f32(sc, so + 1, a.dtype, k.o);
    }
  }
}

// ---- whole vectors: D = 16 L dims, L a power of two; a multiple of 16 of them turn
// A wave takes a token's heads, 64 / L at a time (queries, then keys, then
// values); lane u of a head holds 8 dims of either half of those that turn (u < R /
// 16: dims 8 u .. and R / 2 + 8 u ..) or of the rest, so that both members of a pair
// (i, i + R / 2), or of pairs (2i, 2i + 1), are its own, and
// a row's cos and sin are loaded once for all heads.  The first heads' loads
// are issued before the token's place is looked up (three dependent loads), the
// next heads' before these are stored.
//
// A prompt is bound by HBM: 8 prompts of 2304 to 4096 tokens, 32 + 8 + 8 heads of 128
// dims in bfloat16, 631 MB in and out in 103 us, 6.1 TB/s (a plain copy reaches 6.0 on this
// card); into 4 bits, values wanted, 245 MB in 44 us, 5.5 TB/s.  Loads and stores pass
// the caches where a row is used once: a tenth longer without (4 bits: no difference, so
// only the loads do).  Where fewer dims turn a head is read in shorter runs: 16 thousand
// tokens of the same heads take 68 us where 128 dims turn, 84 where 64 and 96 where 32 do
// (the general kernel, with 24: 726).  A decoding step is bound by its chain of loads: 32 tokens 3.9 us, 13
// sequences of 1 to 5 tokens into 4 bits 5.5 us.
template <typename T>
__device__ __forceinline__ void kv_load8(const char* p, float* v) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = __builtin_nontemporal_load((const f32x4*)p), b = __builtin_nontemporal_load((const f32x4*)(p + 16));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
    const u32x4 w = __builtin_nontemporal_load((const u32x4*)p);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t b = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
      v[e] = std::is_same_v<T, bf16_t> ? bf16_to_f32(b) : f16_to_f32(b);
    }
  }
}
// ONCE: past the caches (a prompt's rows are far more than they hold)
template <typename T, bool ONCE>
__device__ __forceinline__ void kv_store8(char* p, const float* v) {
  if constexpr (sizeof(T) == 4) {
    *(f32x4*)p = (f32x4){v[0], v[1], v[2], v[3]};
    *(f32x4*)(p + 16) = (f32x4){v[4], v[5], v[6], v[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (std::is_same_v<T, bf16_t>)
        w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){v[2 * e], v[2 * e + 1]}, bf16x2));
      else
        w[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){v[2 * e], v[2 * e + 1]}, f16x2));
    }
    if constexpr (ONCE) __builtin_nontemporal_store(w, (u32x4*)p);
    else *(u32x4*)p = w;
  }
}

// combined over the L lanes of a head
template <class Op, int L>
__device__ __forceinline__ float kv_row(float v) {
  const float id = Op::identity;
  if constexpr (L >= 2) v = Op::apply(v, dpp_f32<0xB1, 0xF>(id, v));
  if constexpr (L >= 4) v = Op::apply(v, dpp_f32<0x4E, 0xF>(id, v));
  if constexpr (L >= 8) v = Op::apply(v, dpp_f32<0x141, 0xF>(id, v));
  if constexpr (L >= 16) v = Op::apply(v, dpp_f32<0x140, 0xF>(id, v));
  return v;
}

template <typename T, int L, bool INT4, bool TREE>
__device__ __forceinline__ void kv_append_body(const KvAppendArgs& a) {
  constexpr int D = 16 * L, RPW = 64 / L, SZ = (int)sizeof(T);
  constexpr int DT = SZ == 4 ? DT_F32 : std::is_same_v<T, bf16_t> ? DT_BF16 : DT_F16;
  const int lane = threadIdx.x & 63, u = lane % L, sub = lane / L;
  const long long w = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = (int)(w / a.chunks), chunk = (int)(w % a.chunks);
  if (t >= a.T) return;
  const int slots = a.Hq + 2 * a.Hkv, groups = (slots + RPW - 1) / RPW;
  const bool turns = u < a.R / 16;
  const int from[2] = {turns ? 8 * u : a.R + 8 * (u - a.R / 16), turns ? a.R / 2 + 8 * u : (a.R + D) / 2 + 8 * (u - a.R / 16)};
  const char* qrow = (const char*)a.q + t * a.q_st * SZ;
  const char* krow = (const char*)a.k + t * a.k_st * SZ;
  const char* vrow = (const char*)a.v + t * a.v_st * SZ;
  // a lane past the last head repeats it and stores nothing
  auto load = [&](int g, float (&x)[2][8]) {
    const int s = min(g * RPW + sub, slots - 1);
    const char* p = s < a.Hq ? qrow + s * a.q_sh * SZ
                             : s < a.Hq + a.Hkv ? krow + (s - a.Hq) * a.k_sh * SZ : vrow + (s - a.Hq - a.Hkv) * a.v_sh * SZ;
    kv_load8<T>(p + from[0] * SZ, x[0]);
    kv_load8<T>(p + from[1] * SZ, x[1]);
  };
  float x[2][8];
  load(chunk, x);
  const KvPlace at = kv_place<TREE>(a, t);
  if (at.seq < 0) return;
  float c[8] = {}, s[8] = {};
  if (turns) {
    // half-split: pairs 8 u .. + 7; interleaved: 4 u .. + 3 and R / 4 + 4 u .. + 3
    const int i0 = a.interleaved ? 4 * u : 8 * u, i1 = a.interleaved ? a.R / 4 + 4 * u : 8 * u + 4;
    const long long co = at.pos * a.cos_s, so = at.pos * a.sin_s;
    if (a.table_dtype == DT_F32) {
      const f32x4 c0 = *(const f32x4*)((const float*)a.cos + co + i0), c1 = *(const f32x4*)((const float*)a.cos + co + i1);
      const f32x4 s0 = *(const f32x4*)((const float*)a.sin + so + i0), s1 = *(const f32x4*)((const float*)a.sin + so + i1);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e] = c0[e]; c[4 + e] = c1[e];
        s[e] = s0[e]; s[4 + e] = s1[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[e] = load_as_f32(a.cos, co + i0 + e, DT); c[4 + e] = load_as_f32(a.cos, co + i1 + e, DT);
        s[e] = load_as_f32(a.sin, so + i0 + e, DT); s[4 + e] = load_as_f32(a.sin, so + i1 + e, DT);
      }
    }
  }
  for (int g = chunk; g < groups; g += a.chunks) {
    float next[2][8];
    if (g + a.chunks < groups) load(g + a.chunks, next);
    const int slot = g * RPW + sub;
    const bool is_q = slot < a.Hq, is_v = slot >= a.Hq + a.Hkv;
    const int h = is_q ? slot : is_v ? slot - a.Hq - a.Hkv : slot - a.Hq;
    if (a.R) {
      float y[2][8];
      if (a.interleaved) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            kv_turn(x[v][2 * e], x[v][2 * e + 1], c[4 * v + e], s[4 * v + e], y[v][2 * e], y[v][2 * e + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) kv_turn(x[0][e], x[1][e], c[e], s[e], y[0][e], y[1][e]);
      }
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[v][e] = is_v || !turns ? x[v][e] : y[v][e];
    }
    if (slot < slots && (is_q || (!INT4 && at.page >= 0))) {
      char* p = is_q ? (char*)a.q_out + (t * a.qo_st + h * a.qo_sh) * SZ
                     : is_v ? (char*)a.v_cache + (at.page * a.vc_p + at.row * a.vc_r + h * a.vc_h) * SZ
                            : (char*)a.k_cache + (at.page * a.kc_p + at.row * a.kc_r + h * a.kc_h) * SZ;
      kv_store8<T, !INT4>(p + from[0] * SZ, x[0]);
      kv_store8<T, !INT4>(p + from[1] * SZ, x[1]);
    }
    if constexpr (INT4) {
      if (g * RPW + RPW > a.Hq) {  // (uniform) some lane holds a key or value
        float lo = x[0][0], hi = x[0][0];
        bool nan = false;
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            nan |= x[v][e] != x[v][e];
            lo = fminf(lo, x[v][e]);
            hi = fmaxf(hi, x[v][e]);
          }
        lo = -kv_row<OpMax, L>(-lo);
        hi = kv_row<OpMax, L>(hi);
        const KvScale k = kv_scale(lo, hi, kv_row<OpMax, L>(nan ? 1.0f : 0.0f) != 0.0f, DT);
        int code[2][8];
        uint32_t word[2] = {0, 0};
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            code[v][e] = kv_code(x[v][e], k);
            word[v] |= (uint32_t)code[v][e] << (4 * e);
          }
        if (slot < slots && !is_q) {
          char* out = is_v ? (char*)a.v_out : (char*)a.k_out;
          if (out) {
            out += (is_v ? t * a.vo_st + h * a.vo_sh : t * a.ko_st + h * a.ko_sh) * SZ;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[v][e] = kv_value(code[v][e], k);
              kv_store8<T, false>(out + from[v] * SZ, x[v]);
            }
          }
          if (at.page >= 0) {
            char* dst = is_v ? (char*)a.v_cache + (at.page * a.vc_p + at.row * a.vc_r + h * a.vc_h)
                             : (char*)a.k_cache + (at.page * a.kc_p + at.row * a.kc_r + h * a.kc_h);
            *(uint32_t*)(dst + from[0] / 2) = word[0];
            *(uint32_t*)(dst + from[1] / 2) = word[1];
            if (u == 0) {
              char* sc = is_v ? (char*)a.v_scale + 2 * (at.page * a.vs_p + at.row * a.vs_r + h * a.vs_h)
                              : (char*)a.k_scale + 2 * (at.page * a.ks_p + at.row * a.ks_r + h * a.ks_h);
              uint32_t pair;
              if constexpr (DT == DT_BF16)
                pair = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){k.s, k.o}, bf16x2));
              else
                pair = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){k.s, k.o}, f16x2));
              *(uint32_t*)sc = pair;
            }
          }
        }
      }
    }
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[v][e] = next[v][e];
  }
}

}  // namespace g950

extern "C" __global__ __launch_bounds__(256) void g950_kv_append_general(const g950::KvAppendArgs a) {
  g950::kv_append_general_body<false>(a);
}
extern "C" __global__ __launch_bounds__(256) void g950_kv_append_tree_general(const g950::KvAppendArgs a) {
  g950::kv_append_general_body<true>(a);
}

#define G950_KV(TNAME, T, D)                                                                             \
  extern "C" __global__ __launch_bounds__(256) void g950_kv_append_##TNAME##_d##D(const g950::KvAppendArgs a) { \
    g950::kv_append_body<T, D / 16, false, false>(a);                                                    \
  }
#define G950_KVT(TNAME, T, D)                                                                                 \
  extern "C" __global__ __launch_bounds__(256) void g950_kv_append_tree_##TNAME##_d##D(const g950::KvAppendArgs a) { \
    g950::kv_append_body<T, D / 16, false, true>(a);                                                          \
  }
#define G950_KV4(TNAME, T, D)                                                                                 \
  extern "C" __global__ __launch_bounds__(256) void g950_kv_append_int4_##TNAME##_d##D(const g950::KvAppendArgs a) { \
    g950::kv_append_body<T, D / 16, true, false>(a);                                                          \
  }
#define G950_KV_SET(M, TNAME, T) \
  M(TNAME, T, 32)                \
  M(TNAME, T, 64)                \
  M(TNAME, T, 128)               \
  M(TNAME, T, 256)
G950_KV_SET(G950_KV, f32, float)
G950_KV_SET(G950_KV, bf16, g950::bf16_t)
G950_KV_SET(G950_KV, f16, g950::f16_t)
G950_KV_SET(G950_KV4, bf16, g950::bf16_t)
G950_KV_SET(G950_KV4, f16, g950::f16_t)
G950_KV_SET(G950_KVT, f32, float)
G950_KV_SET(G950_KVT, bf16, g950::bf16_t)
G950_KV_SET(G950_KVT, f16, g950::f16_t)
