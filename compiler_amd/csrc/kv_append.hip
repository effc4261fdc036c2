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
//   s = T((max - min) / 15), o = T(min + 8 s), c = clamp(rint((x - o) / s) + 8, 0, 15)
// and stands for (c - 8) s + o; T is the model's type.  Byte i holds dims 2i
// (low half) and 2i + 1.  A row whose spread rounds to nothing has s = 0 and o = its value; a row that holds NaN or
// infinities (or whose spread passes fp32) has s = o = NaN.
//
// Nothing is written for tokens past cu[B] or of a sequence whose rows are not
// rows of q; nor, at a position below 0 or past the tables; a page that the
// table or the pool does not hold drops only the cache row.
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

__device__ __forceinline__ KvPlace kv_place(const KvAppendArgs& a, int t) {
  KvPlace w;
  w.pos = w.row = 0;
  w.page = -1;
  int b0 = 0, b1 = 0;
  w.seq = __builtin_amdgcn_readfirstlane(kv_sequence(a.cu, a.B, a.T, t, b0, b1));
  if (w.seq < 0) return w;
  const long long pos = (long long)a.used[w.seq] - (b1 - b0) + (t - b0);
  if (pos < 0 || (a.R && pos >= a.positions)) {
    w.seq = -1;
    return w;
  }
  w.pos = __builtin_amdgcn_readfirstlane((int)pos);
  const int e = w.pos / a.block_size;
  w.row = w.pos % a.block_size;
  if (e < a.max_pages) {
    const int ph = a.table[(long long)w.seq * a.table_s + e];
    w.page = ph >= 0 && ph < a.pages ? ph : -1;
  }
  w.page = __builtin_amdgcn_readfirstlane(w.page);
  return w;
}

// (a, b) turned; each operation rounds on its own
__device__ __forceinline__ void kv_turn(float a, float b, float c, float s, float& y, float& z) {
#pragma clang fp contract(off)
  const float ac = a * c, bs = b * s, bc = b * c, as = a * s;
  y = ac - bs;
  z = bc + as;
}

// an fp32 value as it stands: a following conversion to float16 does not draw
// the operation before it into one rounding (v_fma_mixlo_f16)
__device__ __forceinline__ float kv_keep(float v) {
  asm("" : "+v"(v));
  return v;
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
#pragma clang fp contract(off)
  const float c = rintf((x - k.o) * k.inv) + 8.0f;  // (NaN: 0)
  return (int)fminf(fmaxf(c, 0.0f), 15.0f);
}
__device__ __forceinline__ float kv_value(int c, const KvScale& k) {
  return kv_keep(fmaf((float)(c - 8), k.s, k.o));  // the product is exact
}

// One wave per (token, head) row: any D, R, stride and alignment.
__device__ __forceinline__ void kv_append_general_body(const KvAppendArgs& a) {
  const int lane = threadIdx.x & 63;
  const int slots = a.Hq + 2 * a.Hkv;
  const long long tasks = (long long)a.T * slots;
  const int isz = a.dtype == DT_F32 ? 4 : 2;
  for (long long task = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); task < tasks; task += (long long)gridDim.x * 4) {
    const int t = __builtin_amdgcn_readfirstlane((int)(task / slots));
    const int slot = __builtin_amdgcn_readfirstlane((int)(task % slots));
    const KvPlace w = kv_place(a, t);
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

}  // namespace g950

extern "C" __global__ __launch_bounds__(256) void g950_kv_append_general(const g950::KvAppendArgs a) {
  g950::kv_append_general_body(a);
}
