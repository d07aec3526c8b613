// Low-rank adapters beside a projection, an adapter to a row, and their gradients.  For the rows t of adapter g:
//   s[t] = x[t] . down[g]^T                       out[t] = y[t] + scale[g] * s[t] . up[g]^T
//   gs[t] = scale[g] * gout[t] . up[g]            gx[t] = gs[t] . down[g]
//   gdown[g] = sum_t gs[t]^T x[t]                 gup[g] = scale[g] * sum_t gout[t]^T s[t]
// Sums are in fp32.  s and gs enter all products as two bf16 numbers each, the nearest and what it leaves, so that they have 16 bits there:
// rounded to 8 they would add an error of their own, as large as that of the outputs' rounding (49152 rows of 64 adapters: 0.0023 of error
// in the gradients against 64 bits, and 0.0017 so).
//
// Rows of one adapter are worked on in tiles, and one launch does both products of a tile: a cluster of one to eight blocks splits the
// first over its inner size and the second over its outputs, and joins s through distributed shared memory, always in the blocks' order.
// What has to be moved is x, y and out once and each adapter once; a tile of few rows is bound by the latency of its two chains of copies,
// one of many by the bytes.
#include "tc.cuh"

namespace mg {

namespace {

constexpr int kAdapterTile = 128;           // rows of a tile of a plan
constexpr int kDirectTile = 16;             // rows of a tile that the kernel finds by itself
constexpr int kAdapterThreads = 256;
static_assert(MG_ADAPTER_DIRECT <= kAdapterThreads, "rows of a call without a plan: one to a thread");

__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// BYTES (16 or 8) of a row from element c on, into shared memory; what lies at `end` or behind arrives as zeros and is not read.  Rows begin on
// 16-byte boundaries.
template <int BYTES>
__device__ __forceinline__ void copy_row(uint32_t to, const uint16_t* row, int c, int end) {
  const int have = min(max(2 * (end - c), 0), BYTES);
  const uint16_t* from = have > 0 ? row + c : row;          // an address inside the row for a copy of nothing
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(have) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(have) : "memory");
}
// 16 bytes of a row, all of them there
__device__ __forceinline__ void copy_whole(uint32_t to, const uint16_t* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
// the first `bytes` of them, zeros behind
__device__ __forceinline__ void copy_part(uint32_t to, const uint16_t* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ void st_shared(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// the sum of four numbers over the blocks of the cluster, in the order of the blocks
__device__ __forceinline__ float4 cluster_sum(uint32_t at, int cs) {
  float4 there[8];
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (c < cs) there[c] = ld_cluster_f32x4(map_to_cta(at, c));
  float4 u = there[0];
#pragma unroll
  for (int c = 1; c < 8; ++c)
    if (c < cs) { u.x += there[c].x; u.y += there[c].y; u.z += there[c].z; u.w += there[c].w; }
  return u;
}
// eight numbers, the second four `next` bytes behind the first, over CS blocks from block `base` on
template <int CS>
__device__ __forceinline__ void cluster_sum8(uint32_t at, uint32_t next, int base, float* v) {
  float4 a[CS], b[CS];
#pragma unroll
  for (int c = 0; c < CS; ++c) {
    const uint32_t there = map_to_cta(at, base + c);
    a[c] = ld_cluster_f32x4(there);
    b[c] = ld_cluster_f32x4(there + next);
  }
#pragma unroll
  for (int c = 1; c < CS; ++c) {
    a[0].x += a[c].x; a[0].y += a[c].y; a[0].z += a[c].z; a[0].w += a[c].w;
    b[0].x += b[c].x; b[0].y += b[c].y; b[0].z += b[c].z; b[0].w += b[c].w;
  }
  v[0] = a[0].x; v[1] = a[0].y; v[2] = a[0].z; v[3] = a[0].w;
  v[4] = b[0].x; v[5] = b[0].y; v[6] = b[0].z; v[7] = b[0].w;
}
__device__ __forceinline__ void st_cluster16(uint32_t addr, const uint4& v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// two numbers as bf16 and what that leaves of them as bf16
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& high, uint32_t& low) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const float2 f = __bfloat1622float2(h);
  // what is not finite has no rest: it would make a NaN of an infinity
  const __nv_bfloat162 l = __floats2bfloat162_rn(isfinite(f.x) ? a - f.x : 0.f, isfinite(f.y) ? b - f.y : 0.f);
  high = *reinterpret_cast<const uint32_t*>(&h);
  low = *reinterpret_cast<const uint32_t*>(&l);
}
// two warps wait for one another
__device__ __forceinline__ void pair_sync(int pair) { asm volatile("bar.sync %0, 64;" ::"r"(pair + 1) : "memory"); }
template <int N>
__device__ __forceinline__ uint32_t word_of(const uint4 (&v)[N], int w) {      // w is a constant wherever this is inlined
  const uint4& u = v[w / 4];
  return w % 4 == 0 ? u.x : w % 4 == 1 ? u.y : w % 4 == 2 ? u.z : u.w;
}
// eight elements of a row of n from column c on
__device__ __forceinline__ void store_row(uint16_t* row, int c, int n, const uint4& v) {
  if (c + 8 <= n) {
    *reinterpret_cast<uint4*>(row + c) = v;
  } else {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < n) row[c + e] = static_cast<uint16_t>(u[e >> 1] >> (16 * (e & 1)));
  }
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                 "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr));
  tc_ld_wait();
}
__device__ __forceinline__ void tc_ld8(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
  tc_ld_wait();
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(r[e]);
}
struct AdapterArgs {
  const uint16_t* x;          // rows of the first product, K elements
  int64_t ldx;
  int K;
  const uint16_t* w1;         // the first product's adapters: [rank][K], or [K][rank] on the way back
  int64_t g1, ld1;
  const uint16_t* w2;         // the second's: [N][rank], or [rank][N]
  int64_t g2, ld2;
  const uint16_t* y;          // rows that the second product is added to; nullptr: none
  int64_t ldy;
  uint16_t* out;
  int64_t ldo;
  int N;                      // 0: no second product
  uint16_t* s;                // [n_rows][2][RP]: s and what that leaves; nullptr: not kept
  const float* scale;         // nullptr: 1
  float factor;
  int rank, n_adapters, n_rows;
  const int32_t* ids;         // a call without a plan
  const int4* tiles;          // adapter (-1: none), first entry of order, rows with it, rows; behind them, the tiles of adapters, all, and the
                              // adapters with rows
  int n_tiles, slots;         // tiles there is room for; blocks that run at once, a multiple of a cluster's
  const int32_t* order;
  int32_t* status;
};

// ---- few rows, without a plan ------------------------------------------------------------------
// Tiles of sixteen rows, which the kernel finds by itself: what counts is the latency and the adapters' bytes.  In us, here and by a plan
// that is made already (making it takes 4 to 5 more), K = N = 4096, rank 16: 1 row 5.8 and 15.7, 32 rows with 64 adapters 7.7 and 19.3,
// 128 rows 15.1 and 29.7, 256 rows 13.9 and 31.2, with 8 adapters 12.5 and 16.6; rank 64, 64 adapters 37.8 and 40.0, 8 adapters 19.5 and 19.9;
// rank 128, 64 adapters 52 and 104, 8 adapters 27.4 and 23.2, 128 rows 23.8 and 23.0, 2048 columns 20.0 and 17.6: level with a plan and its
// making, ahead of them elsewhere.  Beyond 256 rows there is no thread to a row for the search, and the plan's larger tiles read the
// adapters less often.
// 201 rows of 64 adapters, 5120 to 1000 columns, rank 12: 11.4 us for 12 MB; bound by two chains of copy, wait and product with a meeting
// of the cluster between them.
// Operands go through a ring
// that every thread fills for itself, in the layout of its MMA fragments: the inner index of a product may be permuted at will, so a
// thread takes 16 adjacent bytes of a row where the fragment names two and two elements apart, and the outputs' index too, so that it
// ends with 16 adjacent bytes of a row of out.
template <int RP>                                              // the rank, filled up
struct DirectCfg {
  static constexpr int NG = RP == 128 ? 2 : 1, NT = RP / 8 / NG;               // groups of warps over the rank, n tiles of a warp
  static constexpr int V1 = 2 + NT, V2 = 2 + RP / 8;           // 16-byte pieces of a thread and a step: rows and adapters, in either product
  static constexpr int STAGES = RP == 16 ? 4 : RP == 128 ? 2 : 3;              // steps on their way
  static constexpr int PIECES = STAGES * (V1 > V2 ? V1 : V2);
  static constexpr size_t RING = static_cast<size_t>(PIECES) * kAdapterThreads * 16;
  static constexpr size_t SMEM = RING + 2 * kDirectTile * RP * 2;
  static_assert(8 / NG * kDirectTile * RP * 4 <= RING && SMEM <= 224 * 1024, "shared memory");
};

template <int RP>
__global__ void __launch_bounds__(kAdapterThreads, RP <= 32 ? 2 : 1) adapter_direct_kernel(const AdapterArgs a) {
  using C = DirectCfg<RP>;
  constexpr int NT = C::NT, NG = C::NG, KS = RP / 16, KGS = 8 / NG, S = C::STAGES;
  extern __shared__ __align__(16) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem);                                   // between the products: [groups over K][rows][RP]
  uint4* frag = reinterpret_cast<uint4*>(smem + C::RING);                        // s: [high, low part][k step][lane]
  __shared__ int s_rows[kDirectTile];
  __shared__ int s_before[kAdapterThreads / 32], s_first;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i = lane >> 2, q = lane & 3;
  const int cs = static_cast<int>(cluster_size()), cr = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / cs;
  const uint32_t ring = smem_u32(smem) + tid * 16;
  auto piece = [&](int j) { return ring + static_cast<uint32_t>(j) * (kAdapterThreads * 16); };
  // Row `tile` begins a tile if as many rows of its adapter lie before it as whole tiles take; the tile is it and the next ones.
  auto id_of = [&](int r) { const int v = a.ids[r]; return v >= 0 && v < a.n_adapters ? v : -1; };
  const int g = id_of(tile);
  {
    const bool same = tid < a.n_rows && id_of(tid) == g;
    const uint32_t votes = __ballot_sync(0xFFFFFFFFu, same);
    if (lane == 0) s_before[warp] = __popc(votes);
    __syncthreads();
    int before = __popc(votes & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) before += s_before[w];
    if (tid == tile) s_first = before;
    __syncthreads();
    const int first = s_first;
    if (first % kDirectTile != 0) return;              // the whole cluster
    if (same && before >= first && before < first + kDirectTile) s_rows[before - first] = tid;
  }
  int all = 0;
  for (int w = 0; w < kAdapterThreads / 32; ++w) all += s_before[w];
  const int len = min(all - s_first, kDirectTile), live = g >= 0 ? len : 0;
  const float scale = g >= 0 ? a.factor * (a.scale != nullptr ? a.scale[g] : 1.0f) : 0.0f;
  __syncthreads();
  int64_t row_of[2];
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) row_of[hf] = s_rows[min(hf * 8 + i, len - 1)];

  if (live > 0) {
    const int ng = warp % NG, kg = warp / NG;
    const uint16_t* w1 = a.w1 + g * a.g1;
    const uint16_t* xp[2] = {a.x + row_of[0] * a.ldx, a.x + row_of[1] * a.ldx};
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    const int slices = (a.K + 31) / 32, per = (slices + cs - 1) / cs;
    const int lo = cr * per, hi = min(slices, lo + per);
    auto fetch = [&](int stage, int sl) {
      if (sl < hi) {
        const int c = sl * 32 + 8 * q;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) copy_row<16>(piece(stage * C::V1 + hf), xp[hf], c, a.K);
        // eight elements of each of NT rows of w1: row i of the n tiles
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int n = (ng * NT + t) * 8 + i;
          copy_row<16>(piece(stage * C::V1 + 2 + t), w1 + (n < a.rank ? n : 0) * a.ld1, c, n < a.rank ? a.K : 0);
        }
      }
      copies_commit();
    };
#pragma unroll
    for (int k = 0; k < S - 1; ++k) fetch(k, lo + kg + k * KGS);
    int stage = 0;
    for (int sl = lo + kg; sl < hi; sl += KGS) {
      fetch(stage == 0 ? S - 1 : stage - 1, sl + (S - 1) * KGS);
      copies_wait<S - 1>();
      const uint4 u0 = ld_shared(piece(stage * C::V1)), u1 = ld_shared(piece(stage * C::V1 + 1));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 v = ld_shared(piece(stage * C::V1 + 2 + t));
        mma_bf16(acc[t], u0.x, u1.x, u0.y, u1.y, v.x, v.y);
        mma_bf16(acc[t], u0.z, u1.z, u0.w, u1.w, v.z, v.w);
      }
      if (++stage == S) stage = 0;
    }
    copies_wait<0>();
    __syncthreads();                                  // the ring is free: the warps' sums go there
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) red[(kg * kDirectTile + (e >> 1) * 8 + i) * RP + ng * NT * 8 + t * 8 + 2 * q + (e & 1)] = acc[t][e];
    __syncthreads();
    // The sums of this block over its warps, then over the blocks of the cluster, always in the same order; the columns behind the rank
    // and the rows behind the tile's are zeros.
    const float4* parts = reinterpret_cast<const float4*>(red);
    constexpr int QUADS = kDirectTile * RP / 4;
    auto block_sum = [&](int p) {
      float4 v = parts[p];
#pragma unroll
      for (int k = 1; k < KGS; ++k) {
        const float4 w = parts[k * QUADS + p];
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      return v;
    };
    for (int p = tid; p < QUADS; p += kAdapterThreads) reinterpret_cast<float4*>(red)[p] = block_sum(p);
    cluster_sync_all();
    for (int p = tid; p < QUADS; p += kAdapterThreads) {
      const int row = 4 * p / RP, r = 4 * p % RP;
      const float4 u = cluster_sum(smem_u32(parts + p), cs);
      float v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = row < live && r + e < a.rank ? v[e] : 0.f;
      uint2 high, low;
      split_pair(v[0], v[1], high.x, low.x);
      split_pair(v[2], v[3], high.y, low.y);
      // the fragments that hold (row, r) to (row, r + 3): see the copies of w2
      const int fi = row & 7, hf = (row >> 3) & 1, fq = RP == 16 ? r >> 2 : (r & 31) >> 3;
      const int ks = RP == 16 ? 0 : (r >> 5) * 2 + ((r >> 2) & 1);
      uint32_t* f = reinterpret_cast<uint32_t*>(frag + ks * 32 + fi * 4 + fq);
      f[hf] = high.x;
      f[2 + hf] = high.y;
      f[KS * 128 + hf] = low.x;
      f[KS * 128 + 2 + hf] = low.y;
      if (a.s != nullptr && cr == 0 && row < len) {
        uint16_t* kept = a.s + static_cast<int64_t>(s_rows[row]) * (2 * RP) + r;
        *reinterpret_cast<uint2*>(kept) = high;
        *reinterpret_cast<uint2*>(kept + RP) = low;
      }
    }
    cluster_sync_all();                               // the ring is free again, here and in the blocks that have read it
  } else if (a.s != nullptr && cr == 0) {
    for (int p = tid; p < len * RP; p += kAdapterThreads)
      *reinterpret_cast<uint32_t*>(a.s + static_cast<int64_t>(s_rows[p / RP]) * (2 * RP) + 2 * (p % RP)) = 0u;
  }

  const int units = (a.N + 31) / 32, each = (units + cs - 1) / cs, last = min(units, (cr + 1) * each);
  if (live == 0 && a.y == a.out && a.ldy == a.ldo) return;            // after the last barrier of the cluster
  const uint16_t* w2 = a.w2 + (g >= 0 ? g * a.g2 : 0);
  auto fetch = [&](int stage, int unit) {
    if (unit < last) {
      const int c0 = unit * 32;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) copy_row<16>(piece(stage * C::V2 + hf), a.y + row_of[hf] * a.ldy, c0 + 8 * q, hf * 8 + i < len ? a.N : 0);
      if (live > 0)
        // of row 4 i + t of the unit's 32 rows of w2, n tile t's row i: the elements of this thread's fragments
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int col = c0 + 4 * i + t, end = col < a.N ? a.rank : 0;
          const uint16_t* row = w2 + (col < a.N ? col : 0) * a.ld2;
          if (RP == 16) copy_row<8>(piece(stage * C::V2 + 2 + t / 2) + t % 2 * 8, row, 4 * q, end);
          else
#pragma unroll
            for (int p = 0; p < RP / 32; ++p) copy_row<16>(piece(stage * C::V2 + 2 + t * (RP / 32) + p), row, 32 * p + 8 * q, end);
        }
    }
    copies_commit();
  };
  const int unit0 = cr * each + warp;
#pragma unroll
  for (int k = 0; k < S - 1; ++k) fetch(k, unit0 + k * (kAdapterThreads / 32));
  int stage = 0;
  for (int unit = unit0; unit < last; unit += kAdapterThreads / 32) {
    fetch(stage == 0 ? S - 1 : stage - 1, unit + (S - 1) * (kAdapterThreads / 32));
    copies_wait<S - 1>();
    const int c = unit * 32 + 8 * q;
    float acc[4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    if (live > 0) {
      uint4 v[KS * 2];
#pragma unroll
      for (int j = 0; j < KS * 2; ++j) v[j] = ld_shared(piece(stage * C::V2 + 2 + j));
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          const uint4 f = frag[(part * KS + ks) * 32 + lane];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int w = RP == 16 ? t * 2 : (t * (RP / 32) + ks / 2) * 4 + ks % 2 * 2;
            mma_bf16(acc[t], f.x, f.y, f.z, f.w, word_of(v, w), word_of(v, w + 1));
          }
        }
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      if (hf * 8 + i >= len || c >= a.N) continue;
      uint4 v = ld_shared(piece(stage * C::V2 + hf));
      if (live > 0) {
        float o[8];
        unpack8(v, o);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(scale, acc[e & 3][hf * 2 + (e >> 2)], o[e]);          // column 4 * (2q + (e >> 2)) + (e & 3) of the unit
        v = pack8(o);
      }
      store_row(a.out + row_of[hf] * a.ldo, c, a.N, v);
    }
    if (++stage == S) stage = 0;
  }
  copies_wait<0>();
}

// ---- tiles of a plan ---------------------------------------------------------------------------
// 128 rows of one adapter on the accumulator's lanes.  A step is 64 columns of x, or 64 columns of out; its tiles are copied to shared memory as
// the tensor core reads them, a few steps ahead (rows wherever the order says, zeros behind what a row or the rank has).  Eight warps copy
// the first product's, then finish s and the outputs, while four others copy the second product's; one has the products done, into tensor
// memory.  s passes through shared memory in two parts of bf16.  A cluster of up to eight blocks shares a tile where there are few: each sums
// s over its columns of x, then over the blocks for its share of the rows, and hands that to all.
// 8192 rows of 4096 to 4096 columns, rank 64, 8 adapters: 55 us for 210 MB, 3.8 TB/s; 49152 rows of 64 adapters in a buffer of 57344, 2048 to
// 2048, rank 16: 145 us for 670 MB, 4.6 TB/s, the way back 110 us for 440 MB.  Within a turn of all places it streams at what memory gives (296
// tiles of 2048 to 2048: 90 us, 5.2 TB/s, 1184 tiles 5.7); what bounds it is the turn that is not full, and where clusters share tiles their
// meeting, 9 of the 55 us, in which all blocks pause at once.  By MMAs of warps on tiles of 16 rows the first took 88 us.
constexpr int kFinishWarps = 8, kCopyWarps = 4, kTileThreads = 32 * (kFinishWarps + kCopyWarps + 1);
template <int RP>
struct TileCfg {
  static constexpr int BLOCKS = RP <= 64 ? 2 : 1;              // per SM
  static constexpr int STAGES = RP == 64 ? 3 : 4;
  static constexpr int ROWS = kAdapterTile * 128;              // bytes of a stage: the rows' tile, then the adapter's
  static constexpr int STAGE = ROWS + (RP <= 64 ? 8192 : 16384);
  static constexpr int PART = RP <= 32 ? 64 : ROWS * (RP / 64);                  // from one part of s to the other: blocks of 64 columns, or half a row
  static constexpr size_t SMEM = static_cast<size_t>(STAGES) * STAGE + (RP <= 32 ? ROWS : 2 * PART);
  static constexpr int COLS = 256, SECOND = 128;               // of tensor memory; the second product's two accumulators of 64
  static_assert(kAdapterTile * RP * 4 <= (RP <= 32 ? ROWS : 2 * PART) && BLOCKS * (SMEM + 2048) <= 228 * 1024, "shared memory");
};
// operand whose inner index goes over rows of 128 bytes (64 outer elements each), swizzled: 64 outer elements outer_bytes apart
__device__ __forceinline__ uint64_t rows_desc(uint32_t saddr, uint32_t outer_bytes) {
  return (make_smem_desc(saddr) & ~(0x3FFFull << 16)) | static_cast<uint64_t>(outer_bytes >> 4) << 16;
}
__host__ __device__ constexpr uint32_t mma_shape(int n) { return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n) >> 3 << 17) | (8u << 24); }
constexpr uint32_t kRowsA = 1u << 15, kRowsB = 1u << 16;        // operand A, B by rows_desc

// for the tensor core: this warp's copies but those of the last LEFT steps, and what it has written before
template <int LEFT>
__device__ __forceinline__ void arrive(uint64_t* full) {
  copies_wait<LEFT>();
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(full));
}
// What one of WARPS warps' threads copies of a step: 16 bytes of some rows of the tile of rows, 128 bytes of a row side by side (with 64 the load and
// store unit was what 8192 rows of 4096 x 4096 waited for; rows that are not there are the last one again), and pieces of the adapter's tile,
// RP rows of 64 elements (wide) or 64 rows of RP (narrow).
template <int RP, bool BACK, int WARPS>
struct TileCopies {
  using C = TileCfg<RP>;
  static constexpr int ROWS = WARPS * 4, EACH = kAdapterTile / ROWS;             // rows of an instruction of all warps, rows of a thread
  static constexpr int PIECES = RP * 8 / (WARPS * 32) > 0 ? RP * 8 / (WARPS * 32) : 1, NARROW_ROWS = WARPS * 32 / (RP / 8);
  const AdapterArgs& a;
  const uint16_t *wide, *narrow;
  int t;
  const uint16_t* from[EACH];
  __device__ TileCopies(const AdapterArgs& args, int g, int thread) : a(args), t(thread) {
    const uint16_t *w1 = a.w1 + g * a.g1, *w2 = a.w2 + g * a.g2;
    wide = BACK ? w2 : w1;
    narrow = BACK ? w1 : w2;
  }
  __device__ __forceinline__ void rows_of(const uint16_t* base, int64_t ld, const int* rows, int n) {
#pragma unroll
    for (int j = 0; j < EACH; ++j) from[j] = base + static_cast<int64_t>(rows[min((t >> 3) + j * ROWS, n - 1)]) * ld + (t & 7) * 8;
  }
  // into the stage at `to`: columns c to c + 63 of n of the first `rows` rows, and of the adapter
  __device__ __forceinline__ void step(uint32_t to, bool first, int c, int n, int rows) const {
    const int r0 = t >> 3, p = t & 7, first_row = t / 32 * 4;
    const uint32_t mine = r0 * 128 + ((p ^ (r0 & 7)) << 4);
    const bool inside = c + 64 <= n;
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (first_row + j * ROWS < rows) {
        if (inside) copy_whole(to + mine + j * ROWS * 128, from[j] + c);
        else copy_row<16>(to + mine + j * ROWS * 128, from[j] - p * 8, c + p * 8, n);
      }
    if (RP * 8 < WARPS * 32 && t >= RP * 8) return;
    if (first != BACK) {
      const int64_t ld = BACK ? a.ld2 : a.ld1;
      if (inside) {
        const uint16_t *first_row = wide + p * 8 + c, *w = first_row + r0 * ld;
#pragma unroll
        for (int j = 0; j < PIECES; ++j, w += ROWS * ld) {
          const bool there = r0 + j * ROWS < a.rank;
          copy_part(to + C::ROWS + mine + j * ROWS * 128, there ? w : first_row, there ? 16 : 0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const int r = r0 + j * ROWS;
          copy_row<16>(to + C::ROWS + mine + j * ROWS * 128, wide + (r < a.rank ? r : 0) * ld, c + p * 8, r < a.rank ? n : 0);
        }
      }
    } else {
      const int64_t ld = BACK ? a.ld1 : a.ld2;
      const int nr = t / (RP / 8), np = t % (RP / 8);
      const uint32_t at = to + C::ROWS + (np >> 3) * 8192 + nr * 128 + (((np & 7) ^ (nr & 7)) << 4);
      if (inside) {
        const int bytes = min(max(2 * (a.rank - np * 8), 0), 16);
        const uint16_t* w = narrow + (c + nr) * ld + (bytes > 0 ? np * 8 : 0);
#pragma unroll
        for (int j = 0; j < PIECES; ++j, w += NARROW_ROWS * ld) copy_part(at + j * NARROW_ROWS * 128, w, bytes);
      } else {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const int r = c + nr + j * NARROW_ROWS;
          copy_row<16>(at + j * NARROW_ROWS * 128, narrow + (r < n ? r : 0) * ld, np * 8, r < n ? a.rank : 0);
        }
      }
    }
  }
};

// The rows of a tile none of which has an adapter: out = y, and s zeros, or gx zeros; columns lo to hi of each.  A warp to a row, 4 KB of it at a
// time.
template <int RP, bool BACK>
__device__ __forceinline__ void rows_without(const AdapterArgs& a, const int32_t* order, int len, int lo, int hi, bool first) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool in_place = !BACK && a.y == a.out && a.ldy == a.ldo;
  for (int r = warp; r < len; r += kTileThreads / 32) {
    const int64_t row = order[r];
    if (!BACK && a.s != nullptr && first)              // gs is read for rows with an adapter only
      for (int p = lane; p < RP / 4; p += 32) reinterpret_cast<uint4*>(a.s + row * (2 * RP))[p] = make_uint4(0u, 0u, 0u, 0u);
    if (in_place) continue;
    uint16_t* to = a.out + row * a.ldo;
    const uint16_t* from = BACK ? nullptr : a.y + row * a.ldy;
    for (int c = lo + lane * 8; c < hi; c += 8 * 32 * 8) {
      uint4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = make_uint4(0u, 0u, 0u, 0u);
        if (!BACK && c + k * 256 + 8 <= hi) v[k] = *reinterpret_cast<const uint4*>(from + c + k * 256);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k * 256 + 8 <= hi) *reinterpret_cast<uint4*>(to + c + k * 256) = v[k];
    }
    const int rest = hi & ~7;                          // hi is the rows' end where it is not a multiple of 8
    if (lo < hi && rest + lane < hi) to[rest + lane] = BACK ? static_cast<uint16_t>(0) : from[rest + lane];
  }
}

template <int RP, bool BACK>
__global__ void __launch_bounds__(kTileThreads, TileCfg<RP>::BLOCKS) adapter_tile_kernel(const AdapterArgs a) {
  using C = TileCfg<RP>;
  constexpr int S = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t s_full[S], s_done[S], s_empty[S], s_first, s_ready;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ int s_rows[kAdapterTile];
  const uint32_t ring = smem_u32(smem_raw), s_at = ring + S * C::STAGE;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // The blocks of a cluster, 2^most of them, share a tile among cs, or take one each.  Tiles of adapters that fill all places take one each; the
  // rest of them are shared by as many as let them all run at once; then come those of rows without an adapter, shared by P.
  const int most = 31 - __clz(cluster_size()), P = 1 << most, pr = static_cast<int>(cluster_ctarank()), cl = blockIdx.x >> most;
  const int4 total = a.tiles[a.n_tiles];
  int4 guess[4];                                       // the tile if there is no full round, by 1, 2, 4 and 8 blocks, on its way beside the numbers
#pragma unroll
  for (int k = 0; k < 4; ++k) guess[k] = a.tiles[min((cl << most >> k) + (pr >> k), a.n_tiles - 1)];
  const int solo = total.x / a.slots * a.slots, rem = total.x - solo;
  int by = most;
  while (by > 0 && rem << by > a.slots) --by;
  const int c1 = solo >> most, c2 = c1 + (((rem << by) + P - 1) >> most);
  const int shift = cl < c1 ? 0 : cl < c2 ? by : a.N > 0 ? most : 0;
  const int first = cl < c1 ? 0 : cl < c2 ? c1 : c2, before = cl < c1 ? 0 : cl < c2 ? solo : total.x;
  const int tile = before + ((cl - first) << most >> shift) + (pr >> shift), end = cl < c2 ? (cl < c1 ? solo : total.x) : total.y;
  const int cs = 1 << shift, cr = pr & (cs - 1), base = pr - cr;
  auto meet = [&]() {                                  // who has nothing to share meets the others of its cluster all the same
    for (int k = 0; cs > 1 && cl < c2 && k < 3; ++k) cluster_sync_all();
  };
  int4 job = make_int4(-1, 0, 0, 0);
  if (tile < end) {
    if (solo == 0 && cl < c2) {
      job = guess[0];
#pragma unroll
      for (int k = 1; k < 4; ++k)
        if (shift == k) job = guess[k];
    } else {
      job = a.tiles[tile];
    }
  }
  const int g = job.x, live = job.z, len = job.w;
  const int units = (a.N + 63) / 64, each = (units + cs - 1) / cs;
  const int lo2 = cr * each, n2 = max(min(units, lo2 + each) - lo2, 0);
  if (live == 0) {
    if (len > 0) rows_without<RP, BACK>(a, a.order + job.y, len, lo2 * 64, min(a.N, (lo2 + n2) * 64), cr == 0);
    meet();
    return;
  }
  if (tid < len) s_rows[tid] = a.order[job.y + tid];
  if (tid == 0) {
    for (int k = 0; k < S; ++k) {
      mbar_init(smem_u32(&s_full[k]), kFinishWarps);
      mbar_init(smem_u32(&s_done[k]), 1);
      mbar_init(smem_u32(&s_empty[k]), kFinishWarps);
    }
    mbar_init(smem_u32(&s_first), 1);
    mbar_init(smem_u32(&s_ready), kFinishWarps);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kFinishWarps + kCopyWarps) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(C::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int slices = (a.K + 63) / 64, per = (slices + cs - 1) / cs;
  const int lo1 = cr * per, n1 = max(min(slices, lo1 + per) - lo1, 0);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // Steps are numbered through both products; step k fills stage k % S for the k / S-th time, and the m-th of the second product empties its stage
  // for the m / S-th.
  auto full = [&](int k) { return wait_warp(smem_u32(&s_full[k % S]), (k / S) & 1, &s_abort, a.status, 120); };
  auto done = [&](int k) { return wait_warp(smem_u32(&s_done[k % S]), (k / S) & 1, &s_abort, a.status, 121); };
  auto empty = [&](int m) { return wait_warp(smem_u32(&s_empty[(n1 + m) % S]), (m / S) & 1, &s_abort, a.status, 122); };

  if (warp == kFinishWarps + kCopyWarps) {
    // ---- products ----
    for (int k = 0; k < n1; ++k) {
      full(k);
      tc_fence_after();
      if (elect_one()) {
        const uint32_t at = ring + k % S * C::STAGE;
        const uint64_t da = make_smem_desc(at), db = BACK ? rows_desc(at + C::ROWS, 8192) : make_smem_desc(at + C::ROWS);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          tc_mma_bf16(tmem, da + 2 * j, db + (BACK ? 128 : 2) * j, mma_shape(RP) | (BACK ? kRowsB : 0u), k + j > 0 ? 1u : 0u);
        tc_commit(smem_u32(&s_done[k % S]));
        if (k == n1 - 1) tc_commit(smem_u32(&s_first));          // for who has not waited for every phase before
      }
      __syncwarp();
    }
    if (cs > 1)
      for (int k = 0; k < 3; ++k) cluster_sync_all();
    wait_warp(smem_u32(&s_ready), 0, &s_abort, a.status, 123);
    for (int m = 0; m < n2; ++m) {
      full(n1 + m);
      if (m >= 2) empty(m - 2);                        // the accumulator has been read
      tc_fence_after();
      if (elect_one()) {
        const uint32_t at = ring + (n1 + m) % S * C::STAGE + C::ROWS, d = tmem + C::SECOND + (m & 1) * 64;
        const uint64_t da = make_smem_desc(s_at), db = BACK ? rows_desc(at, 8192) : make_smem_desc(at);
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int k = 0; k < RP / 16; ++k)
            tc_mma_bf16(d, da + (part * C::PART + (k >> 2) * C::ROWS) / 16 + 2 * (k & 3), db + (BACK ? 128 * k : (k >> 2) * 512 + 2 * (k & 3)),
                        mma_shape(64) | (BACK ? kRowsB : 0u), part + k > 0 ? 1u : 0u);
        tc_commit(smem_u32(&s_done[(n1 + m) % S]));
      }
      __syncwarp();
    }
  } else if (warp >= kFinishWarps) {
    // ---- copies of the second product, from step n1 + S - 1 on ----
    TileCopies<RP, BACK, kCopyWarps> copies(a, g, tid - kFinishWarps * 32);
    if (!BACK) copies.rows_of(a.y, a.ldy, s_rows, len);
    if (n1 > 0) wait_warp(smem_u32(&s_first), 0, &s_abort, a.status, 126);       // the first product has left its last stage
    bool met = cs == 1;
    for (int m = S - 1; m < n2 + S - 2; ++m) {
      if (m >= S && !met) {                            // the blocks' exchange, which comes before any stage is emptied
        for (int k = 0; k < 3; ++k) cluster_sync_all();
        met = true;
      }
      if (m < n2) {
        if (m >= S) empty(m - S);
        copies.step(ring + (n1 + m) % S * C::STAGE, false, (lo2 + m) * 64, a.N, BACK ? 0 : len);
      }
      copies_commit();
      copies_wait<S - 2>();                            // step m - (S - 2) is there, for the tensor core too
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (m >= 2 * S - 3 && lane < kFinishWarps / kCopyWarps) mbar_arrive(smem_u32(&s_full[(n1 + m - (S - 2)) % S]));
    }
    if (!met)
      for (int k = 0; k < 3; ++k) cluster_sync_all();
  } else {
    // ---- s, and the outputs ----
    // A lane finishes a row, 64 bytes to a warp, so that two warps share 32 rows; each stores 16 of them, 128 bytes of a row side by side.
    const int quarter = warp & 3, side = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const float scale = a.factor * (a.scale != nullptr ? a.scale[g] : 1.0f);
    const bool in_place = a.y == a.out && a.ldy == a.ldo;
    {
      // ---- copies of the first product and of the second's first S - 1 steps ----
      TileCopies<RP, BACK, kFinishWarps> copies(a, g, tid);
      if (n1 > 0) copies.rows_of(a.x, a.ldx, s_rows, live);
      auto fetch = [&](int k) {
        if (k < n1) {
          copies.step(ring + k % S * C::STAGE, true, (lo1 + k) * 64, a.K, live);
        } else if (k < n1 + n2) {
          if (!BACK && k == n1) copies.rows_of(a.y, a.ldy, s_rows, len);
          copies.step(ring + k % S * C::STAGE, false, (lo2 + k - n1) * 64, a.N, BACK ? 0 : len);
        }
        copies_commit();
      };
#pragma unroll 1
      for (int k = 0; k < S - 1; ++k) fetch(k);
      for (int k = 0; k < n1; ++k) {
        arrive<S - 2>(&s_full[k % S]);
        if (k > 0) done(k - 1);
        fetch(k + S - 1);
      }
      if (n1 > 0) done(n1 - 1);
    }
    // eight columns of a row of s, zeros behind the tile's rows and the rank, in two parts
    auto parts = [&](int r, int col, float* v, uint4& high, uint4& low) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = r < live && col + e < a.rank ? (BACK ? scale * v[e] : v[e]) : 0.f;
      split_pair(v[0], v[1], high.x, low.x);
      split_pair(v[2], v[3], high.y, low.y);
      split_pair(v[4], v[5], high.z, low.z);
      split_pair(v[6], v[7], high.w, low.w);
      if (a.s != nullptr && r < len) {
        uint16_t* kept = a.s + static_cast<int64_t>(s_rows[r]) * (2 * RP) + col;
        *reinterpret_cast<uint4*>(kept) = high;
        *reinterpret_cast<uint4*>(kept + RP) = low;
      }
      return s_at + (col >> 6) * C::ROWS + r * 128;
    };
    auto low_piece = [&](int r, int col) { return (((RP <= 32 ? 4 : 0) + (col >> 3 & 7)) ^ (r & 7)) << 4; };      // in the second part's row
    tc_fence_after();
    // the accumulator's row of this thread, half of the columns to either side's warps
#pragma unroll
    for (int k = 0; k < RP / 2; k += 8) {
      float v[8];
      const int col = side * (RP / 2) + k;
      tc_ld8(lanes + col, v);
      if (n1 == 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      if (cs == 1) {
        uint4 high, low;
        const uint32_t to = parts(row, col, v, high, low);
        st_shared(to + (((col >> 3 & 7) ^ (row & 7)) << 4), high);
        st_shared(to + (RP <= 32 ? 0 : C::PART) + low_piece(row, col), low);
      } else {                                       // [groups of four columns][row], where s will be
#pragma unroll
        for (int e = 0; e < 2; ++e)
          st_shared(s_at + ((col / 4 + e) * kAdapterTile + row) * 16,
                    make_uint4(__float_as_uint(v[4 * e]), __float_as_uint(v[4 * e + 1]), __float_as_uint(v[4 * e + 2]), __float_as_uint(v[4 * e + 3])));
      }
    }
    if (cs > 1) {
      constexpr int ITEMS = RP <= 32 ? 1 : RP / 32;
      const int share = kAdapterTile / cs;
      float v[ITEMS][8];
      cluster_sync_all();                            // the blocks' sums are there
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) {
        const int q = tid + n * kFinishWarps * 32, r = cr * share + q % share, col = q / share * 8;
        const uint32_t at = s_at + (col / 4 * kAdapterTile + r) * 16;
        if (q >= share * RP / 8) continue;
        if (cs == 8) cluster_sum8<8>(at, kAdapterTile * 16, base, v[n]);
        else if (cs == 4) cluster_sum8<4>(at, kAdapterTile * 16, base, v[n]);
        else cluster_sum8<2>(at, kAdapterTile * 16, base, v[n]);
      }
      cluster_sync_all();                            // and have been read: s takes their place
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) {
        const int q = tid + n * kFinishWarps * 32, r = cr * share + q % share, col = q / share * 8;
        if (q >= share * RP / 8) continue;
        uint4 high, low;
        const uint32_t to = parts(r, col, v[n], high, low);
        for (int c = 0; c < cs; ++c) {                // every block begins with itself
          const uint32_t there = map_to_cta(to, base + ((cr + c) & (cs - 1)));
          st_cluster16(there + (((col >> 3 & 7) ^ (r & 7)) << 4), high);
          st_cluster16(there + (RP <= 32 ? 0 : C::PART) + low_piece(r, col), low);
        }
      }
      asm volatile("fence.proxy.async;" ::: "memory");
      cluster_sync_all();
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&s_ready));
    const int first_row = quarter * 32 + side * 16, piece = lane & 7;
    uint16_t* op[4];
    uint32_t stored = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = first_row + j * 4 + (lane >> 3);
      op[j] = a.out + static_cast<int64_t>(s_rows[min(r, len - 1)]) * a.ldo + piece * 8;
      stored |= (r < len && !(in_place && r >= live) ? 1u : 0u) << j;
    }
#pragma unroll
    for (int k = 0; k < S - 1; ++k)
      if (k < n2) arrive<0>(&s_full[(n1 + k) % S]);
    for (int m = 0; m < n2; ++m) {
      const uint32_t at = ring + (n1 + m) % S * C::STAGE;
      const int c0 = (lo2 + m) * 64;
      full(n1 + m);
      done(n1 + m);
      tc_fence_after();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t acc[16];
        tc_ld16(lanes + C::SECOND + (m & 1) * 64 + side * 32 + h * 16, acc);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t to = at + row * 128 + (((side * 4 + h * 2 + k) ^ (row & 7)) << 4);
          float o[8];
          if (!BACK) unpack8(ld_shared(to), o);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float v = __uint_as_float(acc[8 * k + e]);
            o[e] = BACK ? v : fmaf(scale, v, o[e]);
          }
          if (row < live) st_shared(to, pack8(o));
          else if (BACK) st_shared(to, make_uint4(0u, 0u, 0u, 0u));
        }
      }
      tc_fence_before();
      pair_sync(quarter);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 v = ld_shared(at + (first_row + j * 4 + (lane >> 3)) * 128 + ((piece ^ (lane >> 3) ^ ((j & 1) << 2)) << 4));
        if (stored >> j & 1u) store_row(op[j] + c0, 0, a.N - c0 - piece * 8, v);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s_empty[(n1 + m) % S]));
    }
  }
  tc_fence_before();
  __syncthreads();                                     // other blocks reach for this one's memory between their joint barriers only
  if (warp == kFinishWarps + kCopyWarps) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
  }
}

// ---- gradients of the adapters ---------------------------------------------------------------
// Both are W[c][r] = sum over an adapter's rows t of wide[t][c] * narrow[t][r]: rows of gout and s, of x and gs.  A job is 128 columns c of one
// adapter, on the accumulator's lanes, for all of the rank; a block goes through its rows 64 at a time, then to its next job, whose first
// copies are on their way meanwhile.  Where there are few jobs a cluster's blocks take the steps of one in turn, and their sums meet in a
// fixed order.  The inner index is the rows', so both operands are read as they lie.  The narrow rows' two parts are columns side by side,
// whose sums are added at the end.
// 49152 rows of 64 adapters, 2048 and 2048 columns, rank 16: 77 us for 410 MB, 5.3 TB/s; a job's end, its last product and its sums on their
// way out, is what the SM's other blocks do not quite cover.  Rank 128: 139 us, the narrow rows, twice the wide ones' bytes, from L2.  A job is
// one block's, or one cluster's by the mean number of rows: all 49152 rows on one of 64 adapters take 530 us, loads of 1 / n 148.
struct AdapterGradArgs {
  const uint16_t* wide[2];
  int64_t ldw[2];
  int cols[2], blocks[2];       // columns, and blocks of 128 of them
  const uint16_t* narrow[2];    // [n_rows][2][RP]
  uint16_t* out[2];             // [adapters][cols][rank], [adapters][rank][cols]
  const float* scale;
  float factor;
  int rank, n_adapters, jobs;
  const int4* segs;             // first entry of order, rows and number of every adapter, those of most rows first
  const int4* total;            // .z of them have rows
  const int32_t* order;
  int32_t* status;
};

constexpr int kGradThreads = kAdapterThreads + 32;
// DEEP: two blocks to an SM in the place of three, each with a step more on its way, where no more than two come to an SM anyway.  us, so and
// with three: 65536 rows of one adapter, 2048 and 2048 columns, rank 16 103 and 139; 49152 rows of 64 adapters 84 and 77.
template <int RP, bool DEEP>
struct GradCfg {
  static constexpr int BLOCKS = RP <= 32 && !DEEP ? 3 : 2, STAGES = RP <= 32 ? (DEEP ? 4 : 3) : RP <= 64 ? 3 : 2;
  static constexpr int NR = 2 * RP, HALVES = NR <= 64 ? 1 : NR / 64;             // columns of a narrow row, in blocks of 64
  static constexpr int WIDE = 16384;                           // bytes of a stage: two blocks of 64 columns by 64 rows, then the narrow rows
  static constexpr int STAGE = WIDE + HALVES * 8192;
  static constexpr size_t SMEM = static_cast<size_t>(STAGES) * STAGE + 1024;
  static constexpr int COLS = NR;                              // of tensor memory
  static_assert(128 * RP * 4 <= STAGES * STAGE && BLOCKS * (SMEM + 1536) <= 227 * 1024, "shared memory");
};

// ONE: a job to a block (to a cluster), else one of every gridDim.x
template <int RP, bool ONE, bool DEEP>
__global__ void __launch_bounds__(kGradThreads, GradCfg<RP, DEEP>::BLOCKS) adapter_grad_kernel(const AdapterGradArgs a) {
  using C = GradCfg<RP, DEEP>;
  constexpr int S = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t s_full[S], s_done[S];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quarter = warp & 3, side = warp >> 2;
  const int cs = ONE ? static_cast<int>(cluster_size()) : 1, cr = ONE ? static_cast<int>(cluster_ctarank()) : 0;
  struct Job {
    int g, c0, start, live, steps;                     // steps: of this block, cr, cr + cs, ...
    bool which;
  };
  auto job_of = [&](int n) {
    Job j;
    const int per = a.blocks[0] + a.blocks[1];
    const int at = n / per, block = n - at * per;
    j.which = block >= a.blocks[0];
    j.c0 = (block - (j.which ? a.blocks[0] : 0)) * 128;
    const int4 seg = a.segs[at];
    j.start = seg.x;
    j.live = seg.y;
    j.g = seg.z;
    const int all = (seg.y + 63) / 64;
    j.steps = cr < all ? (all - cr + cs - 1) / cs : 0;
    return j;
  };
  const int with_rows = ONE ? 0 : a.total->z;
  const int first = ONE ? static_cast<int>(blockIdx.x) / cs : static_cast<int>(blockIdx.x);
  const int last = ONE ? first + 1 : with_rows * (a.blocks[0] + a.blocks[1]);
  // the jobs' lengths descend: turns go to and fro, the last block of one being the first of the next
  const int both = 2 * static_cast<int>(gridDim.x), hop0 = ONE ? 1 : both - 1 - 2 * first;
  if (tid == 0) {
    for (int k = 0; k < S; ++k) { mbar_init(smem_u32(&s_full[k]), kAdapterThreads / 32); mbar_init(smem_u32(&s_done[k]), 1); }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(C::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  if (warp == 8) {
    int k = 0;
    for (int n = first, hop = hop0; n < last; n += hop, hop = both - hop) {
      const int steps = job_of(n).steps;
      for (int i = 0; i < steps; ++i, ++k) {
        wait_warp(smem_u32(&s_full[k % S]), (k / S) & 1, &s_abort, a.status, 127);       // a job's first: also that the accumulator has been read
        tc_fence_after();
        if (elect_one()) {
          const uint32_t at = ring + k % S * C::STAGE;
          const uint64_t da = rows_desc(at, 8192), db = rows_desc(at + C::WIDE, 8192);
#pragma unroll
          for (int j = 0; j < 4; ++j) tc_mma_bf16(tmem, da + 128 * j, db + 128 * j, mma_shape(C::NR) | kRowsA | kRowsB, i + j > 0 ? 1u : 0u);
          tc_commit(smem_u32(&s_done[k % S]));
        }
        __syncwarp();
      }
    }
  } else {
    const int r0 = tid >> 3, p = tid & 7;              // this thread's 16 bytes of rows r0 and r0 + 32, of 128 bytes each
    const uint32_t mine = r0 * 128 + ((p ^ (r0 & 7)) << 4);
    // the next step to fetch: its job, its number in it, its rows
    int ahead = first, ahead_hop = hop0, in = 0, rows[2];
    Job f = job_of(first);
    uint32_t filling = ring;
    auto look = [&]() {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int t = (cr + in * cs) * 64 + j * 32 + r0;
        rows[j] = in < f.steps && t < f.live ? a.order[f.start + t] : -1;
      }
    };
    auto next_job = [&]() {
      ahead += ahead_hop;
      ahead_hop = both - ahead_hop;
      if (ahead < last) f = job_of(ahead);
      in = 0;
    };
    look();
    auto fetch = [&]() {                               // what lies behind the last row or column arrives as zeros
      if (ONE ? in < f.steps : ahead < last) {
        const int cols = f.which ? a.cols[1] : a.cols[0], c = f.c0 + p * 8;
        const uint16_t* wide = f.which ? a.wide[1] : a.wide[0];
        const uint16_t* narrow = f.which ? a.narrow[1] : a.narrow[0];
        const int64_t ldw = f.which ? a.ldw[1] : a.ldw[0];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int64_t row = max(rows[j], 0);
          const bool there = rows[j] >= 0;
          const int bytes = there ? 16 : 0;
          const uint16_t* w = wide + row * ldw;
          const uint16_t* n = narrow + row * C::NR + p * 8;
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (f.c0 + 128 <= cols) copy_part(filling + mine + j * 4096 + b * 8192, w + c + b * 64, bytes);
            else copy_row<16>(filling + mine + j * 4096 + b * 8192, w, c + b * 64, there ? cols : 0);
          }
#pragma unroll
          for (int b = 0; b < C::HALVES; ++b)
            if (p < C::NR / 8) copy_part(filling + C::WIDE + mine + j * 4096 + b * 8192, n + b * 64, bytes);
        }
        ++in;
        if (!ONE && in == f.steps) next_job();
        look();
      }
      copies_commit();
      filling = filling == ring + (S - 1) * C::STAGE ? ring : filling + C::STAGE;
    };
    auto done = [&](int k) { wait_warp(smem_u32(&s_done[k % S]), (k / S) & 1, &s_abort, a.status, 128); };
#pragma unroll 1
    for (int k = 0; k < S - 1; ++k) fetch();
    int k = 0;
    for (int n = first, hop = hop0; n < last; n += hop, hop = both - hop) {
      const Job j = job_of(n);
      const int cols = j.which ? a.cols[1] : a.cols[0];
      uint16_t* out = (j.which ? a.out[1] : a.out[0]) + static_cast<int64_t>(j.g) * a.rank * cols;
      for (int i = 0; i < j.steps; ++i, ++k) {
        arrive<S - 2>(&s_full[k % S]);
        if (k > 0) done(k - 1);
        fetch();
      }
      if (ONE && j.live == 0) {
        // zeros, 16 bytes at a time where rows begin so: 128 columns of every one of the rank, or the rank of 128 columns in a piece
        const int have = min(cols - j.c0, 128);
        const int lines = j.which ? a.rank : 1, width = j.which ? have : have * a.rank;
        const int64_t ld = j.which ? cols : 0;
        uint16_t* zeros = out + (j.which ? j.c0 : static_cast<int64_t>(j.c0) * a.rank);
        const bool wide = reinterpret_cast<uintptr_t>(zeros) % 16 == 0 && ld % 8 == 0 && width % 8 == 0;
        const int each = wide ? 8 : 1, pieces = width / each;
        for (int e = cr * kAdapterThreads + tid; e < lines * pieces; e += cs * kAdapterThreads) {
          const int line = lines == 1 ? 0 : e / pieces;
          uint16_t* at = zeros + line * ld + static_cast<int64_t>(e - line * pieces) * each;
          if (wide) *reinterpret_cast<uint4*>(at) = make_uint4(0u, 0u, 0u, 0u);
          else *at = 0;
        }
        continue;
      }
      if (j.steps > 0) done(k - 1);
      tc_fence_after();
      const float scale = j.which ? 1.0f : a.factor * (a.scale != nullptr ? a.scale[j.g] : 1.0f);
      auto store8 = [&](int c, int r, float* v) {      // eight of the rank of one column
        if (c >= cols) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= scale;
        if (!j.which && r + 8 <= a.rank && a.rank % 8 == 0) {
          *reinterpret_cast<uint4*>(out + static_cast<int64_t>(c) * a.rank + r) = pack8(v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (r + e < a.rank)
              out[j.which ? (r + e) * static_cast<int64_t>(cols) + c : static_cast<int64_t>(c) * a.rank + r + e] =
                  __bfloat16_as_ushort(__float2bfloat16_rn(v[e]));
        }
      };
      // a lane a column, half of the rank to either side's warps
      const int col = quarter * 32 + lane;
#pragma unroll
      for (int q = 0; q < RP / 2; q += 8) {
        float v[8];
        const int r = side * (RP / 2) + q;
        float rest[8];
        tc_ld8(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + r, v);
        tc_ld8(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + RP + r, rest);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = isfinite(v[e]) ? v[e] + rest[e] : v[e];       // zeros of the second parts times an infinity are NaN
        if (j.steps == 0)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = 0.f;
        if (cs == 1) {
          store8(j.c0 + col, r, v);
        } else {                                       // [groups of four of the rank][column]
#pragma unroll
          for (int e = 0; e < 2; ++e)
            st_shared(ring + ((r / 4 + e) * 128 + col) * 16,
                      make_uint4(__float_as_uint(v[4 * e]), __float_as_uint(v[4 * e + 1]), __float_as_uint(v[4 * e + 2]), __float_as_uint(v[4 * e + 3])));
        }
      }
      if (cs > 1) {
        cluster_sync_all();
        const int share = 128 / cs;
        for (int q = tid; q < share * RP / 8; q += kAdapterThreads) {
          const int c = cr * share + q % share, r = q / share * 8;
          float v[8];
          const uint32_t at = ring + (r / 4 * 128 + c) * 16;
          if (cs == 8) cluster_sum8<8>(at, 128 * 16, 0, v);
          else if (cs == 4) cluster_sum8<4>(at, 128 * 16, 0, v);
          else cluster_sum8<2>(at, 128 * 16, 0, v);
          store8(j.c0 + c, r, v);
        }
      }
    }
    // the adapters without rows, whose gradients are zeros: 32 KB at a time
#pragma unroll
    for (int which = 0; !ONE && which < 2; ++which) {
      const int64_t size = static_cast<int64_t>(a.rank) * a.cols[which];
      const int chunks = static_cast<int>((size + 16383) / 16384);
      const bool wide = reinterpret_cast<uintptr_t>(a.out[which]) % 16 == 0 && size % 8 == 0;
      if (a.out[which] == nullptr) continue;
      for (int64_t n = blockIdx.x; n < static_cast<int64_t>(a.n_adapters - with_rows) * chunks; n += gridDim.x) {
        const int e = static_cast<int>(n / chunks), part = static_cast<int>(n - static_cast<int64_t>(e) * chunks);
        uint16_t* to = a.out[which] + a.segs[with_rows + e].z * size + static_cast<int64_t>(part) * 16384;
        const int have = static_cast<int>(min(size - static_cast<int64_t>(part) * 16384, static_cast<int64_t>(16384)));
        if (wide)
          for (int q = tid; q < have / 8; q += kAdapterThreads) reinterpret_cast<uint4*>(to)[q] = make_uint4(0u, 0u, 0u, 0u);
        else
          for (int q = tid; q < have; q += kAdapterThreads) to[q] = 0;
      }
    }
    copies_wait<0>();
  }
  if (cs > 1) {                                        // no block leaves while another reads its sums
    if (job_of(first).live > 0 && warp == 8) cluster_sync_all();
    cluster_sync_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS) : "memory");
  }
}

// ---- plans -----------------------------------------------------------------------------------
constexpr int kPlanWarps = 32, kPlanAhead = 8;
struct PlanLayout { int64_t tiles, segs, order, place, words; };          // offsets in words
PlanLayout plan_layout(int64_t rows, int64_t adapters) {
  PlanLayout p;
  // tiles: G groups of rows, some of none, are cut into (rows - G) / 128 + G at most, rounded down; G is adapters + 2 at most
  const int64_t n = (rows + kAdapterTile - 1) / kAdapterTile + adapters + 1;
  p.tiles = 0;
  p.segs = 4 * (n + 1);
  p.order = p.segs + 4 * adapters;
  p.place = p.order + rows;                // while the plan is made
  p.words = p.place + rows;
  return p;
}

// One block sorts the rows by adapter, rows without one last, every adapter's in ascending order, and cuts them into tiles.  Warps take
// runs of rows and count them by adapter; with the counts of the warps before, every row has its place.
// SORTED: the rows lie in segments already (pad_offsets, counts); the order is the rows' own, written by the other blocks.  Each offset counts as
// no less than those in front of it, so that whatever they hold every row is in one tile, those in front of the first segment and behind
// the last among them.
template <bool SORTED>
__global__ void __launch_bounds__(kPlanWarps * 32) adapter_plan_kernel(const int32_t* ids, const int32_t* counts, const int32_t* pad,
                                                                       int rows, int adapters, int n_tiles, int4* tiles, int4* segs,
                                                                       int32_t* order, int32_t* place) {
  extern __shared__ __align__(16) int s_mem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, groups = adapters + (SORTED ? 2 : 1);
  if (SORTED && blockIdx.x > 0) {
    const int64_t at = static_cast<int64_t>(blockIdx.x - 1) * blockDim.x + tid;
    if (at < rows) order[at] = static_cast<int32_t>(at);
    return;
  }
  int* s_start = s_mem;                    // [groups] first entry of order
  int* s_len = s_start + groups;           // rows of the segment
  int* s_live = s_len + groups;            // of which with the adapter
  int* s_tile = s_live + groups;           // [groups + 1] tiles before
  int* s_hist = s_tile + groups + 1;       // [warps][groups]
  auto id_of = [&](int64_t j) {            // -1: no row
    const int v = j < rows ? ids[j] : 0;
    return j < rows ? (v >= 0 && v < adapters ? v : adapters) : -1;
  };
  const int per = ((rows + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const int64_t from = static_cast<int64_t>(warp) * per;
  const bool kept = per <= 32 * kPlanAhead;            // a lane's rows stay in its registers
  int ids_of[kPlanAhead], place_of[kPlanAhead];
  if (!SORTED) {
    for (int e = tid; e < kPlanWarps * groups; e += blockDim.x) s_hist[e] = 0;
    __syncthreads();
    for (int k = 0; k < per; k += 32 * kPlanAhead) {   // the ids of a run on their way together
#pragma unroll
      for (int n = 0; n < kPlanAhead; ++n) ids_of[n] = k + n * 32 < per ? id_of(from + k + n * 32 + lane) : -1;
#pragma unroll
      for (int n = 0; n < kPlanAhead; ++n) {
        if (k + n * 32 >= per) break;
        const int id = ids_of[n];
        const uint32_t peers = __match_any_sync(0xFFFFFFFFu, id);
        const int before = __popc(peers & ((1u << lane) - 1u));
        int at = 0;
        if (id >= 0 && before == 0) {
          at = s_hist[warp * groups + id];
          s_hist[warp * groups + id] = at + __popc(peers);
        }
        at = __shfl_sync(0xFFFFFFFFu, at, __ffs(peers) - 1) + before;
        place_of[n] = at;                              // among the warp's rows of the adapter
        if (!kept && id >= 0) place[from + k + n * 32 + lane] = at;
        __syncwarp();
      }
    }
    __syncthreads();
    for (int e = warp; e < groups; e += kPlanWarps) {  // lane: a warp's count
      const int n = s_hist[lane * groups + e];
      int in = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, in, o);
        if (lane >= o) in += u;
      }
      s_hist[lane * groups + e] = in - n;
      if (lane == 31) {
        s_len[e] = in;
        s_live[e] = e < adapters ? in : 0;
      }
    }
  } else {
    auto clipped = [&](int e) { return min(max(pad[e], 0), rows); };
    bool descends = false;
    for (int e = tid; e <= adapters; e += blockDim.x) {
      const int lo = clipped(e), hi = e < adapters ? clipped(e + 1) : rows;
      s_start[e] = lo;
      s_len[e] = hi - lo;
      s_live[e] = e < adapters ? min(max(counts[e], 0), hi - lo) : 0;
      descends |= hi < lo;
    }
    if (tid == 0) {                                    // in front of the first segment
      s_start[adapters + 1] = 0;
      s_len[adapters + 1] = clipped(0);
      s_live[adapters + 1] = 0;
    }
    // Offsets as they should be are done; a walk over them in any case takes 0.7 of 3.1 us.
    if (__syncthreads_or(descends)) {
      if (warp == 0) {                                 // the largest so far, in runs of a lane
        const int run = (adapters + 32) / 32;
        int most = 0;
        for (int k = 0; k < run; ++k)
          if (lane * run + k <= adapters) most = max(most, s_start[lane * run + k]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xFFFFFFFFu, most, o);
          if (lane >= o) most = max(most, u);
        }
        most = __shfl_up_sync(0xFFFFFFFFu, most, 1);
        if (lane == 0) most = 0;
        for (int k = 0; k < run; ++k)
          if (lane * run + k <= adapters) s_start[lane * run + k] = most = max(most, s_start[lane * run + k]);
      }
      __syncthreads();
      for (int e = tid; e <= adapters; e += blockDim.x) {
        const int len = (e < adapters ? s_start[e + 1] : rows) - s_start[e];
        s_len[e] = len;
        s_live[e] = e < adapters ? min(max(counts[e], 0), len) : 0;
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    const int run = (groups + 31) / 32;
    int n = 0, nt = 0;
    for (int k = 0; k < run; ++k)
      if (lane * run + k < groups) {
        n += s_len[lane * run + k];
        nt += (s_len[lane * run + k] + kAdapterTile - 1) / kAdapterTile;
      }
    int in = n, it = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, in, o), v = __shfl_up_sync(0xFFFFFFFFu, it, o);
      if (lane >= o) { in += u; it += v; }
    }
    in -= n;
    it -= nt;
    for (int k = 0; k < run; ++k) {
      const int e = lane * run + k;
      if (e >= groups) break;
      if (!SORTED) s_start[e] = in;
      s_tile[e] = it;
      in += s_len[e];
      it += (s_len[e] + kAdapterTile - 1) / kAdapterTile;
      if (e == groups - 1) s_tile[groups] = it;
    }
  }
  __syncthreads();
  static_assert(MG_ADAPTER_MAX <= kPlanWarps * 32, "a thread to an adapter");
  int with_rows;
  {                                        // the adapters by their rows: 2^bits neighbouring threads compare one with all
    int bits = 5;
    while (bits > 0 && adapters << bits > kPlanWarps * 32) --bits;
    const int e = tid >> bits, n = e < adapters ? s_live[e] : 0;
    int before = 0;
    if (e < adapters)
      for (int f = tid & ((1 << bits) - 1); f < adapters; f += 1 << bits) before += s_live[f] > n || (s_live[f] == n && f < e);
    for (int o = 1 << bits >> 1; o > 0; o >>= 1) before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
    const bool one = e < adapters && (tid & ((1 << bits) - 1)) == 0;
    if (one) segs[before] = make_int4(s_start[e], n, e, 0);
    with_rows = __syncthreads_count(one && n > 0);
  }
  if (tid == 0) tiles[n_tiles] = make_int4(min(s_tile[adapters], n_tiles), min(s_tile[groups], n_tiles), with_rows, 0);
  for (int e = tid; e < n_tiles; e += blockDim.x) {
    int4 t = make_int4(-1, 0, 0, 0);
    if (e < s_tile[groups]) {
      int lo = 0, hi = groups;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_tile[mid] <= e) lo = mid; else hi = mid;
      }
      const int off = (e - s_tile[lo]) * kAdapterTile;
      const int live = min(max(s_live[lo] - off, 0), kAdapterTile);
      t = make_int4(live > 0 ? lo : -1, s_start[lo] + off, live, min(s_len[lo] - off, kAdapterTile));
    }
    tiles[e] = t;
  }
  if (!SORTED && kept) {
#pragma unroll
    for (int n = 0; n < kPlanAhead; ++n)
      if (n * 32 < per && ids_of[n] >= 0)
        order[s_start[ids_of[n]] + s_hist[warp * groups + ids_of[n]] + place_of[n]] = static_cast<int32_t>(from + n * 32 + lane);
  } else if (!SORTED) {
#pragma unroll 4
    for (int k = 0; k < per; k += 32) {
      const int64_t j = from + k + lane;
      const int id = id_of(j);
      if (id >= 0) order[s_start[id] + s_hist[warp * groups + id] + place[j]] = static_cast<int32_t>(j);
    }
  }
}

int padded_rank(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

template <int RP>
int launch_direct_as(const Handle* h, const AdapterArgs& a, cudaStream_t st) {
  static bool done[64];
  if (int rc = allow_smem(h, adapter_direct_kernel<RP>, DirectCfg<RP>::SMEM, done)) return rc;
  // Blocks to a row's cluster; those whose row begins no tile end at once.  201 rows, us, with 2: 13.3, 4: 11.2, 8: 14.6.
  int cs = 8;
  while (cs > 2 && static_cast<int64_t>(a.n_rows) * cs > 8 * h->sm_count) cs /= 2;
  MG_CUDA(launch_clusters(adapter_direct_kernel<RP>, a.n_rows, cs, kAdapterThreads, DirectCfg<RP>::SMEM, st, a));
  return MG_OK;
}
template <int RP, bool BACK>
int launch_tiles_as(const Handle* h, AdapterArgs a, cudaStream_t st) {
  using C = TileCfg<RP>;
  static bool done[64];
  if (int rc = allow_smem(h, adapter_tile_kernel<RP, BACK>, C::SMEM, done)) return rc;
  // As many blocks to a tile as run at once, were all rows in full tiles; how many tiles there are in earnest the device knows.  K = N = 4096, 8
  // adapters, us with 1, 2, 4, 8 blocks: 1024 rows rank 16 90, 50, 28, 18; 4096 rows 92, 51, 39, 41; 8192 rows rank 64 107, 65, 55, 73; 16384
  // rows rank 16 99, 83, 84, 91; 32768 rows 159, 160, 162, 171.  Elsewhere clusters of four cost: they leave places of a GPC empty, and 296 full
  // tiles of 2048 to 2048 take 123 where single blocks take 90.
  // Rows in not much more than a tile to an adapter, as those of expert-sorted buffers of few tokens, are shared at any number of tiles, since
  // most of them may be without an adapter: by four blocks, or by two where there are many tiles for the length of their rows.  add and
  // grad x, us, by 1, 2 and 4 (tiles, of which with an adapter; K = N):
  //   2048, rank 16:  81, 8: 45 36, 32 25, 32 18    161, 16: 64 43, 43 31, 60 34    258, 25: 74 50, 65 41, 94 58    296, 256: 76 54, 78 59, 89 69
  //   2048, rank 128: 81, 8: 58 45, 39 30, 33 21    161, 16: 68 52, 45 35, 67 43    258, 25: 69 57, 69 47, 104 68
  //   4096, rank 16:  101, 10: 89 72, 67 47, 52 34  165, 80: 120 83, 92 59, 79 63   185, 160: 124 91, 111 90, 114 91   258, 25: 154 95, 118 64, 125 77
  //   7168, rank 16, by 2 and 4: 101, 10: 110 78, 90 55   161, 16: 149 94, 130 70   264, 128: 213 126, 219 138   347, 300: 330 233, 389 283
  const int64_t full = (static_cast<int64_t>(a.n_rows) + kAdapterTile - 1) / kAdapterTile, places = C::BLOCKS * h->sm_count;
  const int least = 4 * full > 5 * a.n_adapters ? 1 : 20 * full > (a.K > a.N ? a.K : a.N) ? 2 : 4;
  int P = 8;
  while (P > least && full * P > places) P /= 2;
  a.slots = static_cast<int>(places / P * P);
  const int64_t all = a.n_tiles + full, most = a.n_tiles + full * P + (P > 1 ? a.slots : 0);      // blocks, P to a tile and one to those of adapters
  // two clusters more: one for what is left of a round, one for rows without an adapter that begin a tile at both ends of the buffer
  MG_CUDA(launch_clusters(adapter_tile_kernel<RP, BACK>, (all * P < most ? all * P : most) / P + 2, P, kTileThreads, C::SMEM, st, a));
  return MG_OK;
}
template <bool BACK>
int launch_tiles(const Handle* h, const AdapterArgs& a, cudaStream_t st) {
  switch (padded_rank(a.rank)) {
    case 16: return launch_tiles_as<16, BACK>(h, a, st);
    case 32: return launch_tiles_as<32, BACK>(h, a, st);
    case 64: return launch_tiles_as<64, BACK>(h, a, st);
    default: return launch_tiles_as<128, BACK>(h, a, st);
  }
}
int launch_direct(const Handle* h, const AdapterArgs& a, cudaStream_t st) {
  switch (padded_rank(a.rank)) {
    case 16: return launch_direct_as<16>(h, a, st);
    case 32: return launch_direct_as<32>(h, a, st);
    case 64: return launch_direct_as<64>(h, a, st);
    default: return launch_direct_as<128>(h, a, st);
  }
}
template <int RP, bool ONE, bool DEEP>
int launch_grad_jobs(const Handle* h, const AdapterGradArgs& a, int64_t clusters, int cs, cudaStream_t st) {
  static bool done[64];
  if (int rc = allow_smem(h, adapter_grad_kernel<RP, ONE, DEEP>, GradCfg<RP, DEEP>::SMEM, done)) return rc;
  MG_CUDA(launch_clusters(adapter_grad_kernel<RP, ONE, DEEP>, clusters, cs, kGradThreads, GradCfg<RP, DEEP>::SMEM, st, a));
  return MG_OK;
}
template <int RP>
int launch_grad_as(const Handle* h, const AdapterGradArgs& a, int cs, cudaStream_t st) {
  // Blocks that stay where there are more jobs than places: the next job's copies are on their way while one ends.  2048 and 2048 columns,
  // 64 adapters, rank 16, us, a job to a block and so: 4 rows each 19.5 and 14.0, 128 rows 27 and 22, 512 rows 55.8 and 52; 768 rows of a
  // skewed routing 79 and 79, if the plan names the adapters of most rows first and the turns go to and fro (in the adapters' order 91 and 122).
  const int most = GradCfg<RP, false>::BLOCKS * h->sm_count;
  if (cs == 1 && a.jobs > most) return launch_grad_jobs<RP, false, false>(h, a, most, 1, st);
  constexpr bool choice = GradCfg<RP, true>::BLOCKS < GradCfg<RP, false>::BLOCKS;
  const bool deep = choice && static_cast<int64_t>(a.jobs) * cs <= 2 * h->sm_count;
  return deep ? launch_grad_jobs<RP, true, choice>(h, a, a.jobs, cs, st) : launch_grad_jobs<RP, true, false>(h, a, a.jobs, cs, st);
}

}  // namespace

int adapter_rank_stride(int rank) { return 2 * padded_rank(rank); }
size_t adapter_plan_bytes(int64_t rows, int64_t adapters) { return static_cast<size_t>(plan_layout(rows, adapters).words) * 4; }

int launch_adapter_plan(const Handle* h, const int32_t* ids, const int32_t* counts, const int32_t* pad, int64_t rows, int adapters,
                        void* plan, cudaStream_t st) {
  const PlanLayout p = plan_layout(rows, adapters);
  int32_t* w = static_cast<int32_t*>(plan);
  const int n_tiles = static_cast<int>(p.segs / 4) - 1, groups = adapters + (ids != nullptr ? 1 : 2);
  static bool done[2][64];
  constexpr size_t most = (4 * (MG_ADAPTER_MAX + 1) + 1 + kPlanWarps * (MG_ADAPTER_MAX + 1)) * sizeof(int);
  const size_t smem = (4 * groups + 1 + (ids != nullptr ? kPlanWarps * groups : 0)) * sizeof(int);
  if (ids != nullptr) {
    if (int rc = allow_smem(h, adapter_plan_kernel<false>, most, done[0])) return rc;
    adapter_plan_kernel<false><<<1, kPlanWarps * 32, smem, st>>>(ids, nullptr, nullptr, static_cast<int>(rows), adapters, n_tiles,
                                                                reinterpret_cast<int4*>(w), reinterpret_cast<int4*>(w + p.segs), w + p.order, w + p.place);
  } else {
    const unsigned blocks = static_cast<unsigned>(1 + (rows + kPlanWarps * 32 - 1) / (kPlanWarps * 32));
    adapter_plan_kernel<true><<<blocks, kPlanWarps * 32, smem, st>>>(nullptr, counts, pad, static_cast<int>(rows), adapters, n_tiles,
                                                                    reinterpret_cast<int4*>(w), reinterpret_cast<int4*>(w + p.segs), w + p.order, w + p.place);
  }
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

static AdapterArgs adapter_args(const Handle* h, const mg_adapters* d, int64_t rows, const int32_t* ids, const void* plan) {
  AdapterArgs a{};
  a.status = h->d_status;
  a.scale = d->d_scale;
  a.factor = d->factor;
  a.rank = d->rank;
  a.n_adapters = d->n_adapters;
  a.n_rows = static_cast<int>(rows);
  if (plan != nullptr) {
    const PlanLayout p = plan_layout(rows, d->n_adapters);
    const int32_t* w = static_cast<const int32_t*>(plan);
    a.tiles = reinterpret_cast<const int4*>(w);
    a.n_tiles = static_cast<int>(p.segs / 4) - 1;
    a.order = w + p.order;
  } else {
    a.ids = ids;
  }
  return a;
}

int launch_adapter_add(const Handle* h, const mg_adapters* d, const void* x, int64_t ldx, const void* y, int64_t ldy, int64_t rows,
                       const int32_t* ids, const void* plan, void* out, int64_t ldo, void* s, cudaStream_t st) {
  AdapterArgs a = adapter_args(h, d, rows, ids, plan);
  a.x = static_cast<const uint16_t*>(x); a.ldx = ldx; a.K = static_cast<int>(d->cols);
  a.w1 = static_cast<const uint16_t*>(d->d_down); a.g1 = d->down_stride; a.ld1 = d->ld_down;
  a.w2 = static_cast<const uint16_t*>(d->d_up); a.g2 = d->up_stride; a.ld2 = d->ld_up;
  a.y = static_cast<const uint16_t*>(y); a.ldy = ldy;
  a.out = static_cast<uint16_t*>(out); a.ldo = ldo; a.N = static_cast<int>(d->n_out);
  a.s = static_cast<uint16_t*>(s);
  return plan != nullptr ? launch_tiles<false>(h, a, st) : launch_direct(h, a, st);
}

int launch_adapter_grad(const Handle* h, const mg_adapters* d, const void* gout, int64_t ldg, const void* x, int64_t ldx, int64_t rows,
                        const void* plan, const void* s, void* gs, void* gx, int64_t ldgx, void* gdown, void* gup, cudaStream_t st) {
  AdapterArgs a = adapter_args(h, d, rows, nullptr, plan);
  a.x = static_cast<const uint16_t*>(gout); a.ldx = ldg; a.K = static_cast<int>(d->n_out);
  a.w1 = static_cast<const uint16_t*>(d->d_up); a.g1 = d->up_stride; a.ld1 = d->ld_up;
  a.w2 = static_cast<const uint16_t*>(d->d_down); a.g2 = d->down_stride; a.ld2 = d->ld_down;
  a.out = static_cast<uint16_t*>(gx); a.ldo = ldgx; a.N = gx != nullptr ? static_cast<int>(d->cols) : 0;
  a.s = static_cast<uint16_t*>(gs);
  if (gx != nullptr || gdown != nullptr)
    if (int rc = launch_tiles<true>(h, a, st)) return rc;
  if (gdown == nullptr && gup == nullptr) return MG_OK;
  AdapterGradArgs b{};
  b.wide[0] = static_cast<const uint16_t*>(gout); b.ldw[0] = ldg; b.cols[0] = static_cast<int>(d->n_out);
  b.narrow[0] = static_cast<const uint16_t*>(s); b.out[0] = static_cast<uint16_t*>(gup);
  b.wide[1] = static_cast<const uint16_t*>(x); b.ldw[1] = ldx; b.cols[1] = static_cast<int>(d->cols);
  b.narrow[1] = static_cast<const uint16_t*>(gs); b.out[1] = static_cast<uint16_t*>(gdown);
  for (int i = 0; i < 2; ++i) b.blocks[i] = b.out[i] != nullptr ? (b.cols[i] + 127) / 128 : 0;
  b.status = h->d_status;
  b.scale = a.scale;
  b.factor = a.factor;
  b.rank = a.rank;
  b.order = a.order;
  b.total = a.tiles + a.n_tiles;
  b.n_adapters = d->n_adapters;
  b.segs = reinterpret_cast<const int4*>(static_cast<const int32_t*>(plan) + plan_layout(rows, d->n_adapters).segs);
  const int64_t jobs = static_cast<int64_t>(d->n_adapters) * (b.blocks[0] + b.blocks[1]);       // below 2^28
  b.jobs = static_cast<int>(jobs);
  // An adapter's rows among several blocks while all of them run at once, two to an SM, and each has two steps, were all adapters alike.
  // 2048 and 2048 columns, us, within 2 blocks to an SM, within 4, within 8: 4096 rows of 4 adapters, rank 16 12.7, 15.3, 22.6; 16384 rows
  // of 8 30.5, 37.1, 39.2; 4096 columns, rank 64 70, 70, 76.
  int cs = 8;
  while (cs > 1 && (rows / d->n_adapters < 128 * cs || jobs * cs > 2 * h->sm_count)) cs /= 2;
  switch (padded_rank(a.rank)) {
    case 16: return launch_grad_as<16>(h, b, cs, st);
    case 32: return launch_grad_as<32>(h, b, cs, st);
    case 64: return launch_grad_as<64>(h, b, cs, st);
    default: return launch_grad_as<128>(h, b, cs, st);
  }
}

}  // namespace mg
