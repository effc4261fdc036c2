// Moving the accepted path of a drafted tree to where its tokens belong in a
// paged cache, on gfx950: cache row base + i gets what row base + path[z, i] held
// (base = used[z] - n, n the tree's nodes), for i < count[z] and i <= path[z, i] < n, whose
// pages the pool holds; every other row is left alone.
//
// A thread owns one piece of a row of one head for the whole path.  A row is
// read (path[i'] >= i' > i) only after the rows before i', all of which lie below it, were
// written or not at all, so taking the path in order, 8 rows at a time, reads every
// row before it is written.
//
// Bound by a launch and a chain of loads (lengths, path, page, rows): 16 paths in one layer of 8
// heads of 128 in bfloat16 take 3.8 us, 32 paths in 16 layers (17 MB read and written, much of it
// in the MALL) 4.6.  Words of 16 bytes where rows, strides and addresses allow, else of 4 or
// single values.
namespace g950 {

template <typename W>
__device__ __forceinline__ void kv_keep_body(const KvKeepArgs& a) {
  const int lane = threadIdx.x & 63;
  // workgroups: pieces of a sequence's rows, then sequences, then layers
  const unsigned blk = blockIdx.x % (unsigned)a.blocks, zl = blockIdx.x / (unsigned)a.blocks;
  const int z = zl % (unsigned)a.B, layer = zl / (unsigned)a.B;
  const int b0 = a.cu[z], b1 = a.cu[z + 1];
  const int n = b0 >= 0 && b1 >= b0 && b1 <= a.T ? b1 - b0 : 0;
  const int count = min(max(a.count[z * a.count_z], 0), min(a.L, n));
  const int used = a.used[z];
  if (blk == 0 && layer == 0 && threadIdx.x == 0) a.used_out[z * a.out_z] = used - n + count;
  const long long base = (long long)used - n;
  const int per = a.words * a.Hkv;  // pieces of a cache row
  const int piece = (int)blk * 256 + threadIdx.x;
  const bool on = piece < 2 * per;
  const bool is_v = piece >= per;
  const int r = is_v ? piece - per : piece, h = r / a.words, w = r % a.words;
  W* cache = (W*)((is_v ? a.v : a.k) + (long long)layer * (is_v ? a.v_l : a.k_l) + (long long)h * (is_v ? a.v_h : a.k_h)) + w;
  const long long sp = is_v ? a.v_p : a.k_p, sr = is_v ? a.v_r : a.k_r;
  auto place = [&](long long row, int& page, int& at) {
    page = -1;
    at = 0;
    if (row < 0) return;
    const long long e = row / a.block_size;
    if (e < a.max_pages) {
      const int ph = a.table[(long long)z * a.table_s + e];
      page = ph < a.pages ? ph : -1;
      at = (int)(row % a.block_size);
    }
  };
  for (int i0 = 0; i0 < count; i0 += 64) {
    // lane i: where row i0 + i comes from and goes to
    const int i = i0 + lane;
    int from = -1, fat = 0, to = -1, tat = 0;
    if (i < count) {
      const int x = a.path[z * a.path_z + i];
      if (x > i && x < n) {
        place(base + x, from, fat);
        place(base + i, to, tat);
      }
    }
    uint64_t todo = __ballot(from >= 0 && to >= 0);
    while (todo) {
      constexpr int U = 8;
      W v[U];
      W* dst[U];
      int m = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        dst[u] = nullptr;
        if (!todo) continue;
        const int l = __ffsll((unsigned long long)todo) - 1;
        todo &= todo - 1;
        m = u + 1;
        const long long src = __builtin_amdgcn_readlane(from, l) * sp + __builtin_amdgcn_readlane(fat, l) * sr;
        dst[u] = (W*)((char*)cache + __builtin_amdgcn_readlane(to, l) * sp + __builtin_amdgcn_readlane(tat, l) * sr);
        if (on) v[u] = *(const W*)((const char*)cache + src);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (on && u < m) *dst[u] = v[u];
    }
  }
}

}  // namespace g950

extern "C" __global__ __launch_bounds__(256) void g950_kv_keep_w16(const g950::KvKeepArgs a) {
  g950::kv_keep_body<g950::u32x4>(a);
}
extern "C" __global__ __launch_bounds__(256) void g950_kv_keep_w4(const g950::KvKeepArgs a) {
  g950::kv_keep_body<uint32_t>(a);
}
extern "C" __global__ __launch_bounds__(256) void g950_kv_keep_w2(const g950::KvKeepArgs a) {
  g950::kv_keep_body<uint16_t>(a);
}
