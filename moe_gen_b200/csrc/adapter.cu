// Low-rank adapters beside a projection, an adapter to a row, and their gradients.  For the rows t of adapter g:
//   s[t] = bf16(x[t] . down[g]^T)                 out[t] = y[t] + scale[g] * s[t] . up[g]^T
//   gs[t] = bf16(scale[g] * gout[t] . up[g])      gx[t] = gs[t] . down[g]
//   gdown[g] = sum_t gs[t]^T x[t]                 gup[g] = scale[g] * sum_t gout[t]^T s[t]
// Sums are in fp32; s and gs are rounded to bf16, the type that the matrix instructions take and that an adapter of bf16 modules
// has between its two products.
//
// Rows of one adapter are worked on in tiles, by the plan's order.  One launch does both products of a tile: a cluster of one to
// eight blocks splits the first product over its inner size and the second over its outputs, and joins s through distributed
// shared memory.  Operands go from global memory into registers in the layout of the MMA's fragments: the inner index of a product
// may be permuted at will, so a thread takes 16 adjacent bytes of a row where the fragment names two and two elements apart, and
// the outputs' index too, so that it ends with 16 adjacent bytes of a row of out.
#include "tc.cuh"

namespace mg {

namespace {

constexpr int kAdapterTile = 64;            // rows of a tile of a plan
constexpr int kDirectTile = 16;             // rows of a tile that the kernel finds by itself
constexpr int kDirectRows = 256;            // rows of a call without a plan, at most: one to a thread
constexpr int kAdapterThreads = 256;

__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t lows(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t highs(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
// rows that are read once: not kept in L1, where the adapters are
__device__ __forceinline__ uint4 ld_once(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// W 32-bit words of a row from element c on; what lies at `end` or behind is 0 and not read.  Rows begin on 16-byte boundaries.
template <int W>
__device__ __forceinline__ void load_words(const uint16_t* row, int c, int end, uint32_t* v) {
  if (c + 2 * W <= end) {
    if (W == 1) v[0] = __ldg(reinterpret_cast<const uint32_t*>(row + c));
    else if (W == 2) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + c));
      v[0] = u.x; v[W - 1] = u.y;
    } else {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(row + c));
      v[0] = u.x; v[1 % W] = u.y; v[2 % W] = u.z; v[3 % W] = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      v[i] = 0u;
      if (c + 2 * i < end) v[i] = __ldg(row + c + 2 * i);
      if (c + 2 * i + 1 < end) v[i] |= static_cast<uint32_t>(__ldg(row + c + 2 * i + 1)) << 16;
    }
  }
}
__device__ __forceinline__ uint4 load_tail(const uint16_t* row, int c, int end) {
  uint32_t v[4];
  load_words<4>(row, c, end, v);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

// BYTES of a row from element c on, into shared memory; what lies at `end` or behind arrives as zeros and is not read.  Rows begin on
// 16-byte boundaries.
template <int BYTES>
__device__ __forceinline__ void copy_row(uint32_t to, const uint16_t* row, int c, int end) {
  const int have = min(max(2 * (end - c), 0), BYTES);
  const uint16_t* from = have > 0 ? row + c : row;          // an address inside the row for a copy of nothing
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(have) : "memory");
  else if (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(have) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(have) : "memory");
}
// BYTES of a row, all of them there
template <int BYTES>
__device__ __forceinline__ void copy_whole(uint32_t to, const uint16_t* from) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else if (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
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
  uint16_t* s;                // [n_rows][RP]; nullptr: not kept
  const float* scale;         // nullptr: 1
  float factor;
  int rank, n_adapters, n_rows;
  const int32_t* ids;         // a call without a plan
  const int4* tiles;          // adapter (-1: none), first entry of order, rows with it, rows
  const int32_t* order;
};

// NT: n tiles of a warp in the first product, NG: groups of warps over the rank.  BACK: the gradient's two products, whose adapters
// are transposed.
template <int NT, int NG>
struct AdapterCfg {
  static constexpr int RP = NT * NG * 8;                       // the rank, filled up
  static constexpr int V1 = 8 + NT, V2 = 8 + RP / 8;           // 16-byte pieces of a thread and a step: rows and adapters, in either product
  static constexpr int BLOCKS = NT >= 8 ? 1 : 2;               // per SM
  static constexpr int S1 = NT >= 8 ? 3 : 2, S2 = RP == 64 ? 3 : 2;        // steps on their way
  static constexpr int PIECES = S1 * V1 > S2 * V2 ? S1 * V1 : S2 * V2;
  static constexpr size_t RING = static_cast<size_t>(PIECES) * kAdapterThreads * 16;
  static constexpr size_t SMEM = RING + kAdapterTile * RP * 2;
  static_assert(8 / NG * kAdapterTile * RP * 4 <= RING && BLOCKS * (SMEM + 2048) <= 227 * 1024, "shared memory");
};

template <int NT, int NG, bool BACK>
__global__ void __launch_bounds__(kAdapterThreads, AdapterCfg<NT, NG>::BLOCKS) adapter_kernel(const AdapterArgs a) {
  using C = AdapterCfg<NT, NG>;
  constexpr int RP = C::RP, KS = RP / 16, KGS = 8 / NG, MT = kAdapterTile / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem);                                   // between the products: [groups over K][rows][RP]
  uint4* frag = reinterpret_cast<uint4*>(smem + C::RING);                        // s: [m tile][k step][lane]
  __shared__ int s_rows[kAdapterTile];
  __shared__ int s_before[kAdapterThreads / 32], s_first;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i = lane >> 2, q = lane & 3;
  const int cs = static_cast<int>(cluster_size()), cr = static_cast<int>(cluster_ctarank());
  const int tile = blockIdx.x / cs;
  // A thread copies what it reads itself: piece j of a stage of V lies beside the other threads' piece j, and it waits for its own copies
  // only.
  const uint32_t ring = smem_u32(smem) + tid * 16;
  auto piece = [&](int j) { return ring + static_cast<uint32_t>(j) * (kAdapterThreads * 16); };
  int g, live, len;
  if (a.tiles != nullptr) {
    const int4 t = a.tiles[tile];
    g = t.x; live = t.z; len = t.w;
    if (len == 0) return;
    if (tid < len) s_rows[tid] = a.order[t.y + tid];
    __syncthreads();
  } else {
    // Row `tile` begins a tile if as many rows of its adapter lie before it as whole tiles take; the tile is it and the next ones.
    auto id_of = [&](int r) { const int v = a.ids[r]; return v >= 0 && v < a.n_adapters ? v : -1; };
    g = id_of(tile);
    const bool same = tid < a.n_rows && id_of(tid) == g;
    const uint32_t votes = __ballot_sync(0xFFFFFFFFu, same);
    if (lane == 0) s_before[warp] = __popc(votes);
    __syncthreads();
    int before = __popc(votes & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < kAdapterThreads / 32; ++w) {
      if (w < warp) before += s_before[w];
      all += s_before[w];
    }
    if (tid == tile) s_first = before;
    __syncthreads();
    const int first = s_first;
    if (first % kDirectTile != 0) return;
    len = min(all - first, kDirectTile);
    live = g >= 0 ? len : 0;
    if (same && before >= first && before < first + len) s_rows[before - first] = tid;
    __syncthreads();
  }
  const float scale = g >= 0 ? a.factor * (a.scale != nullptr ? a.scale[g] : 1.0f) : 0.0f;
  const int live_mts = (live + 15) / 16;

  if (live > 0) {
    const int ng = warp % NG, kg = warp / NG;
    const uint16_t* w1 = a.w1 + g * a.g1 + (BACK ? 0 : static_cast<int64_t>(ng * NT * 8 + i) * a.ld1);
    const uint16_t* xp[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) xp[m][hf] = a.x + static_cast<int64_t>(s_rows[min(m * 16 + hf * 8 + i, live - 1)]) * a.ldx;
    float acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][t][e] = 0.f;
    const int slices = (a.K + 31) / 32, per = (slices + cs - 1) / cs;
    const int lo = cr * per, hi = min(slices, lo + per);
    const bool filled = a.rank == RP;
    auto fetch = [&](int stage, int sl) {
      const int c = sl * 32 + 8 * q;
      if (sl < hi && filled && sl * 32 + 32 <= a.K) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (m < live_mts)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) copy_whole<16>(piece(stage * C::V1 + m * 2 + hf), xp[m][hf] + c);
        const uint16_t* w = BACK ? w1 + c * a.ld1 + ng * NT * 8 + i * NT : w1 + c;
        const int64_t next = BACK ? a.ld1 : 8 * a.ld1;
#pragma unroll
        for (int r = 0; r < (BACK ? 8 : NT); ++r, w += next) {
          if (!BACK) copy_whole<16>(piece(stage * C::V1 + 8 + r), w);
          else copy_whole<NT * 2>(piece(stage * C::V1 + 8 + r * NT / 8) + r * NT % 8 * 2, w);
        }
      } else if (sl < hi) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (m < live_mts)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) copy_row<16>(piece(stage * C::V1 + m * 2 + hf), xp[m][hf], c, a.K);
        if (!BACK) {
          // eight elements of each of NT rows of w1: row i of the n tiles
#pragma unroll
          for (int t = 0; t < NT; ++t)
            copy_row<16>(piece(stage * C::V1 + 8 + t), (ng * NT + t) * 8 + i < a.rank ? w1 + t * 8 * a.ld1 : a.w1, c,
                         (ng * NT + t) * 8 + i < a.rank ? a.K : 0);
        } else {
          // NT elements of each of eight rows of w1: element i * NT + t is row i of n tile t
#pragma unroll
          for (int r = 0; r < 8; ++r)
            copy_row<NT * 2>(piece(stage * C::V1 + 8 + r * NT / 8) + r * NT % 8 * 2, w1 + static_cast<int64_t>(min(c + r, a.K - 1)) * a.ld1,
                             ng * NT * 8 + i * NT, c + r < a.K ? a.rank : 0);
        }
      }
      copies_commit();
    };
#pragma unroll
    for (int k = 0; k < C::S1 - 1; ++k) fetch(k, lo + kg + k * KGS);
    int stage = 0;
    for (int sl = lo + kg; sl < hi; sl += KGS) {
      fetch(stage == 0 ? C::S1 - 1 : stage - 1, sl + (C::S1 - 1) * KGS);
      copies_wait<C::S1 - 1>();
      uint32_t bv[NT * 4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 v = ld_shared(piece(stage * C::V1 + 8 + t));
        bv[4 * t] = v.x; bv[4 * t + 1] = v.y; bv[4 * t + 2] = v.z; bv[4 * t + 3] = v.w;
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= live_mts) break;
        const uint4 u0 = ld_shared(piece(stage * C::V1 + m * 2)), u1 = ld_shared(piece(stage * C::V1 + m * 2 + 1));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          uint32_t b[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t r0 = bv[BACK ? 2 * e * (NT / 2) + t / 2 : 0], r1 = bv[BACK ? (2 * e + 1) * (NT / 2) + t / 2 : 0];
            b[e] = !BACK ? bv[t * 4 + e] : t % 2 ? highs(r0, r1) : lows(r0, r1);
          }
          mma_bf16(acc[m][t], u0.x, u1.x, u0.y, u1.y, b[0], b[1]);
          mma_bf16(acc[m][t], u0.z, u1.z, u0.w, u1.w, b[2], b[3]);
        }
      }
      if (++stage == C::S1) stage = 0;
    }
    copies_wait<0>();
    __syncthreads();                                  // the ring is free: the warps' sums go there
    const int rows = live_mts * 16;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= live_mts) break;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = 2 * q + (e & 1);
          const int r = ng * NT * 8 + (BACK ? n * NT + t : t * 8 + n);
          red[(kg * rows + m * 16 + (e >> 1) * 8 + i) * RP + r] = acc[m][t][e];
        }
    }
    __syncthreads();
    // The sums of this block over its warps, then over the blocks of the cluster, always in the same order; the columns behind the rank
    // and the rows behind the tile's are zeros.
    const float4* parts = reinterpret_cast<const float4*>(red);
    const int quads = rows * RP / 4;
    auto block_sum = [&](int p) {
      float4 v = parts[p];
#pragma unroll
      for (int k = 1; k < KGS; ++k) {
        const float4 u = parts[k * quads + p];
        v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
      }
      return v;
    };
    if (cs > 1) {
      for (int p = tid; p < quads; p += kAdapterThreads) reinterpret_cast<float4*>(red)[p] = block_sum(p);
      cluster_sync_all();
    }
    for (int p = tid; p < quads; p += kAdapterThreads) {
      const int row = 4 * p / RP, r = 4 * p % RP;
      float4 u;
      if (cs > 1) {
        const uint32_t at = smem_u32(parts + p);
        float4 there[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c < cs) there[c] = ld_cluster_f32x4(map_to_cta(at, c));
        u = there[0];
#pragma unroll
        for (int c = 1; c < 8; ++c)
          if (c < cs) { u.x += there[c].x; u.y += there[c].y; u.z += there[c].z; u.w += there[c].w; }
      } else {
        u = block_sum(p);
      }
      float v[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = row < live && r + e < a.rank ? (BACK ? scale * v[e] : v[e]) : 0.f;
      const __nv_bfloat162 b0 = __floats2bfloat162_rn(v[0], v[1]), b1 = __floats2bfloat162_rn(v[2], v[3]);
      const uint2 words = make_uint2(*reinterpret_cast<const uint32_t*>(&b0), *reinterpret_cast<const uint32_t*>(&b1));
      // the fragments that hold (row, r) to (row, r + 3): see the loads of w2 below
      const int fi = row & 7, hf = (row >> 3) & 1, fq = RP == 16 ? r >> 2 : (r & 31) >> 3;
      const int ks = RP == 16 ? 0 : (r >> 5) * 2 + ((r >> 2) & 1);
      uint32_t* f = reinterpret_cast<uint32_t*>(frag + ((row >> 4) * KS + ks) * 32 + fi * 4 + fq);
      f[hf] = words.x;
      f[2 + hf] = words.y;
      if (a.s != nullptr && cr == 0 && row < len) *reinterpret_cast<uint2*>(a.s + static_cast<int64_t>(s_rows[row]) * RP + r) = words;
    }
    if (cs > 1) cluster_sync_all();                   // the ring is free again, here and in the blocks that have read it
    else __syncthreads();
  }
  if (a.s != nullptr && cr == 0) {                    // rows without an adapter
    const int from = live_mts * 16;
    for (int p = tid; p < (len - from) * RP / 2; p += kAdapterThreads)
      *reinterpret_cast<uint32_t*>(a.s + static_cast<int64_t>(s_rows[from + 2 * p / RP]) * RP + 2 * p % RP) = 0u;
  }

  const int units = (a.N + 31) / 32, each = (units + cs - 1) / cs, last = min(units, (cr + 1) * each);
  const int mts = (len + 15) / 16;
  const bool in_place = a.y == a.out && a.ldy == a.ldo;
  const uint16_t* w2 = a.w2 + (g >= 0 ? g * a.g2 : 0);
  const uint16_t* yp[MT][2];
  uint16_t* op[MT][2];                                // nullptr: not written
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int r = m * 16 + hf * 8 + i;
      const int64_t row = s_rows[min(r, len - 1)];
      yp[m][hf] = a.y + row * a.ldy;
      op[m][hf] = r < len && !(in_place && r >= live) ? a.out + row * a.ldo : nullptr;
    }
  const bool filled = a.rank == RP;
  auto fetch = [&](int stage, int unit) {
    const int c0 = unit * 32, c = c0 + 8 * q;
    if (unit < last && filled && c0 + 32 <= a.N) {
      if (a.y != nullptr)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (m < mts)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) copy_whole<16>(piece(stage * C::V2 + m * 2 + hf), yp[m][hf] + c);
      if (live > 0 && !BACK) {
        const uint16_t* w = w2 + (c0 + 4 * i) * a.ld2 + (RP == 16 ? 4 : 8) * q;
#pragma unroll
        for (int t = 0; t < 4; ++t, w += a.ld2) {
          if (RP == 16) copy_whole<8>(piece(stage * C::V2 + 8 + t / 2) + t % 2 * 8, w);
          else
#pragma unroll
            for (int p = 0; p < RP / 32; ++p) copy_whole<16>(piece(stage * C::V2 + 8 + t * (RP / 32) + p), w + 32 * p);
        }
      } else if (live > 0) {
#pragma unroll
        for (int k = 0; k < KS; k += 2) {
          const uint16_t* w = w2 + (RP == 16 ? 4 * q : k * 16 + 8 * q) * a.ld2 + c0 + 4 * i;
#pragma unroll
          for (int e = 0; e < (RP == 16 ? 4 : 8); ++e, w += a.ld2) copy_whole<8>(piece(stage * C::V2 + 8 + k * 2 + e / 2) + e % 2 * 8, w);
        }
      }
    } else if (unit < last) {
      if (a.y != nullptr)
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (m < mts)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) copy_row<16>(piece(stage * C::V2 + m * 2 + hf), yp[m][hf], c, a.N);
      if (live > 0) {
        if (!BACK) {
          // of row 4 i + t of the unit's 32 rows of w2, n tile t's row i: the elements of this thread's fragments
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int col = c0 + 4 * i + t, end = col < a.N ? a.rank : 0;
            const uint16_t* row = w2 + (col < a.N ? col : 0) * a.ld2;
            if (RP == 16) {
              copy_row<8>(piece(stage * C::V2 + 8 + t / 2) + t % 2 * 8, row, 4 * q, end);
            } else {
#pragma unroll
              for (int p = 0; p < RP / 32; ++p) copy_row<16>(piece(stage * C::V2 + 8 + t * (RP / 32) + p), row, 32 * p + 8 * q, end);
            }
          }
        } else {
          // four columns, of n tiles 0 to 3, of the rows of w2 that this thread's fragments hold
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = (RP == 16 ? 4 * q : (ks >> 1) * 32 + 8 * q + (ks & 1) * 4) + e;
              copy_row<8>(piece(stage * C::V2 + 8 + ks * 2 + e / 2) + e % 2 * 8, w2 + (r < a.rank ? r : 0) * a.ld2, c0 + 4 * i,
                          r < a.rank ? a.N : 0);
            }
        }
      }
    }
    copies_commit();
  };
  const int unit0 = cr * each + warp;
#pragma unroll
  for (int k = 0; k < C::S2 - 1; ++k) fetch(k, unit0 + k * (kAdapterThreads / 32));
  int stage = 0;
  for (int unit = unit0; unit < last; unit += kAdapterThreads / 32) {
    fetch(stage == 0 ? C::S2 - 1 : stage - 1, unit + (C::S2 - 1) * (kAdapterThreads / 32));
    copies_wait<C::S2 - 1>();
    const int c = unit * 32 + 8 * q;
    uint32_t b[KS][4][2];
    if (live > 0) {
      uint32_t v[KS * 8];
#pragma unroll
      for (int j = 0; j < KS * 2; ++j) {
        const uint4 u = ld_shared(piece(stage * C::V2 + 8 + j));
        v[4 * j] = u.x; v[4 * j + 1] = u.y; v[4 * j + 2] = u.z; v[4 * j + 3] = u.w;
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            if (!BACK)
              b[ks][t][p] = RP == 16 ? v[t * 2 + p] : v[(t * (RP / 32) + ks / 2) * 4 + ks % 2 * 2 + p];
            else {
              const uint32_t r0 = v[ks * 8 + p * 4 + t / 2], r1 = v[ks * 8 + p * 4 + 2 + t / 2];
              b[ks][t][p] = t % 2 ? highs(r0, r1) : lows(r0, r1);
            }
          }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m >= mts) break;
      float acc[4][4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
      if (m < live_mts) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint4 f = frag[(m * KS + ks) * 32 + lane];
#pragma unroll
          for (int t = 0; t < 4; ++t) mma_bf16(acc[t], f.x, f.y, f.z, f.w, b[ks][t][0], b[ks][t][1]);
        }
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        if (op[m][hf] == nullptr || c >= a.N) continue;
        uint4 v = a.y != nullptr ? ld_shared(piece(stage * C::V2 + m * 2 + hf)) : make_uint4(0u, 0u, 0u, 0u);
        if (m * 16 + hf * 8 + i < live) {
          float o[8];
          unpack8(v, o);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = acc[e & 3][hf * 2 + (e >> 2)];                        // column 4 * (2q + (e >> 2)) + (e & 3) of the unit
            o[e] = BACK ? p : fmaf(scale, p, o[e]);
          }
          v = pack8(o);
        }
        uint16_t* dst = op[m][hf] + c;
        if (c + 8 <= a.N) {
          *reinterpret_cast<uint4*>(dst) = v;
        } else {
          const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < a.N) dst[e] = static_cast<uint16_t>(u[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
    if (++stage == C::S2) stage = 0;
  }
}

// ---- gradients of the adapters ---------------------------------------------------------------
// Both are W[c][r] = sum over an adapter's rows of wide[t][c] * narrow[t][r]: rows of gout and s, of x and gs.  A block holds 256
// columns of one adapter for all of the rank and goes through the rows, which a cluster's blocks take in turn; the sums meet in
// shared memory in a fixed order.  The wide rows are read once.
struct AdapterGradArgs {
  const uint16_t* wide[2];
  int64_t ldw[2];
  int cols[2], blocks[2];       // columns, and blocks of 256 of them
  const uint16_t* narrow[2];    // [n_rows][RP]
  uint16_t* out[2];             // [adapters][cols][rank], [adapters][rank][cols]; nullptr: not wanted
  const float* scale;
  float factor;
  int rank;
  const int2* segs;             // first entry of order and rows of every adapter
  const int32_t* order;
};

template <int NT, int NG>
__global__ void __launch_bounds__(kAdapterThreads, NT >= 8 ? 1 : 2) adapter_grad_kernel(const AdapterGradArgs a) {
  constexpr int RP = NT * NG * 8, PITCH = RP + 1, RGS = 2 / NG;
  extern __shared__ __align__(16) uint8_t smem[];
  float* buf = reinterpret_cast<float*>(smem);       // [256 columns][PITCH]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i = lane >> 2, q = lane & 3;
  const int cs = static_cast<int>(cluster_size()), cr = static_cast<int>(cluster_ctarank());
  const int job = blockIdx.x / cs, per = a.blocks[0] + a.blocks[1];
  const int g = job / per, which = job % per >= a.blocks[0], cb = job % per - (which ? a.blocks[0] : 0);
  const int2 seg = a.segs[g];
  const int live = seg.y, cols = which ? a.cols[1] : a.cols[0];
  const int cg = warp & 3, other = warp >> 2, ng = NG == 2 ? other : 0, rg = NG == 2 ? 0 : other;
  const int c = cb * 256 + cg * 64 + i * 8, r0 = ng * NT * 8 + i * NT;
  const uint16_t* wide = which ? a.wide[1] : a.wide[0];
  const uint16_t* narrow = which ? a.narrow[1] : a.narrow[0];
  const int64_t ldw = which ? a.ldw[1] : a.ldw[0];
  float acc[4][NT][4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][t][e] = 0.f;
  const int step = RGS * cs * 16;
  auto row_of = [&](int t) { return t < live ? a.order[seg.x + t] : -1; };
  int rows[4];
  int t0 = (rg + RGS * cr) * 16;
#pragma unroll
  for (int e = 0; e < 4; ++e) rows[e] = row_of(t0 + 4 * q + e);
  for (; t0 < live; t0 += step) {
    uint4 v[4];
    uint32_t w[4][NT / 2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t row = rows[e];
      v[e] = make_uint4(0u, 0u, 0u, 0u);
      if (row >= 0) v[e] = c + 8 <= cols ? ld_once(wide + row * ldw + c) : load_tail(wide + row * ldw, c, cols);
      load_words<NT / 2>(narrow + (row >= 0 ? row : 0) * RP, r0, row >= 0 ? RP : 0, w[e]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) rows[e] = row_of(t0 + step + 4 * q + e);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t b0 = t % 2 ? highs(w[0][t / 2], w[1][t / 2]) : lows(w[0][t / 2], w[1][t / 2]);
      const uint32_t b1 = t % 2 ? highs(w[2][t / 2], w[3][t / 2]) : lows(w[2][t / 2], w[3][t / 2]);
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        auto word = [m](const uint4& u) { return m == 0 ? u.x : m == 1 ? u.y : m == 2 ? u.z : u.w; };
        const uint32_t x0 = word(v[0]), x1 = word(v[1]), x2 = word(v[2]), x3 = word(v[3]);
        mma_bf16(acc[m][t], lows(x0, x1), highs(x0, x1), lows(x2, x3), highs(x2, x3), b0, b1);
      }
    }
  }
  // row i of m tile m is column 2m of the thread's eight, row i + 8 the one behind it
  auto at = [&](int m, int t, int e) -> float& {
    return buf[(cg * 64 + i * 8 + 2 * m + (e >> 1)) * PITCH + ng * NT * 8 + (2 * q + (e & 1)) * NT + t];
  };
  if (rg == 1)
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) at(m, t, e) = acc[m][t][e];
  __syncthreads();
  if (rg == 0)
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) at(m, t, e) = RGS == 2 ? acc[m][t][e] + at(m, t, e) : acc[m][t][e];
  if (cs > 1) cluster_sync_all();
  else __syncthreads();
  const float scale = which ? 1.0f : a.factor * (a.scale != nullptr ? a.scale[g] : 1.0f);
  uint16_t* out = (which ? a.out[1] : a.out[0]) + static_cast<int64_t>(g) * a.rank * cols;
  const int mine = 256 / cs, first = cr * mine;
  for (int e = tid; e < mine * a.rank; e += kAdapterThreads) {
    const int col = first + (which ? e % mine : e / a.rank), r = which ? e / mine : e % a.rank;
    if (cb * 256 + col >= cols) continue;
    float v = 0.f;
    if (cs > 1) {
      const uint32_t p = smem_u32(buf + col * PITCH + r);
      for (int k = 0; k < cs; ++k) v += ld_cluster_f32(map_to_cta(p, k));
    } else {
      v = buf[col * PITCH + r];
    }
    const int64_t cc = cb * 256 + col;
    out[which ? r * static_cast<int64_t>(cols) + cc : cc * a.rank + r] = __bfloat16_as_ushort(__float2bfloat16_rn(live > 0 ? scale * v : 0.f));
  }
  if (cs > 1) cluster_sync_all();                    // no block leaves while another reads its sums
}

// ---- plans -----------------------------------------------------------------------------------
constexpr int kPlanWarps = 32;
struct PlanLayout { int64_t tiles, segs, order, words; };          // offsets in words
PlanLayout plan_layout(int64_t rows, int64_t adapters) {
  PlanLayout p;
  const int64_t n = (rows + kAdapterTile - 1) / kAdapterTile + adapters + 1;
  p.tiles = 0;
  p.segs = 4 * n;
  p.order = p.segs + 2 * (adapters + (adapters & 1));
  p.words = p.order + rows;
  return p;
}

// One block sorts the rows by adapter, rows without one last, every adapter's in ascending order, and cuts them into tiles.  Warps take
// runs of rows and count them by adapter; with the counts of the warps before, every row has its place.
// SORTED: the rows lie in segments already (pad_offsets, counts); the order is the rows' own, written by the other blocks.
template <bool SORTED>
__global__ void __launch_bounds__(kPlanWarps * 32) adapter_plan_kernel(const int32_t* ids, const int32_t* counts, const int32_t* pad,
                                                                       int rows, int adapters, int n_tiles, int4* tiles, int2* segs,
                                                                       int32_t* order) {
  extern __shared__ __align__(16) int s_mem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, groups = adapters + 1;
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
  const int per = ((rows + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const int64_t from = static_cast<int64_t>(warp) * per;
  if (!SORTED) {
    for (int e = tid; e < kPlanWarps * groups; e += blockDim.x) s_hist[e] = 0;
    __syncthreads();
    for (int k = 0; k < per; k += 32) {
      const int64_t j = from + k + lane;
      const int v = j < rows ? ids[j] : -1;
      const int id = j < rows ? (v >= 0 && v < adapters ? v : adapters) : -1;
      const uint32_t peers = __match_any_sync(0xFFFFFFFFu, id);
      if (id >= 0 && lane == __ffs(peers) - 1) s_hist[warp * groups + id] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    for (int e = tid; e < groups; e += blockDim.x) {
      int run = 0;
      for (int w = 0; w < kPlanWarps; ++w) {
        const int n = s_hist[w * groups + e];
        s_hist[w * groups + e] = run;
        run += n;
      }
      s_len[e] = run;
      s_live[e] = e < adapters ? run : 0;
    }
  } else {
    for (int e = tid; e < groups; e += blockDim.x) {
      const int lo = min(max(pad[e], 0), rows), hi = e < adapters ? min(max(pad[e + 1], lo), rows) : rows;
      s_start[e] = lo;
      s_len[e] = hi - lo;
      s_live[e] = e < adapters ? min(max(counts[e], 0), hi - lo) : 0;
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
  for (int e = tid; e < adapters; e += blockDim.x) segs[e] = make_int2(s_start[e], s_live[e]);
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
  if (!SORTED)
    for (int k = 0; k < per; k += 32) {
      const int64_t j = from + k + lane;
      const int v = j < rows ? ids[j] : -1;
      const int id = j < rows ? (v >= 0 && v < adapters ? v : adapters) : -1;
      const uint32_t peers = __match_any_sync(0xFFFFFFFFu, id);
      const int before = __popc(peers & ((1u << lane) - 1u));
      const int at = id >= 0 ? s_start[id] + s_hist[warp * groups + id] + before : 0;
      __syncwarp();
      if (id >= 0) {
        order[at] = static_cast<int32_t>(j);
        if (before == 0) s_hist[warp * groups + id] += __popc(peers);
      }
      __syncwarp();
    }
}

int padded_rank(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

template <typename... P, typename... A>
cudaError_t launch_clusters(void (*kernel)(P...), int64_t jobs, int cs, size_t smem, cudaStream_t st, A&&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cs;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(jobs * cs));
  cfg.blockDim = dim3(kAdapterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// a kernel's dynamic shared memory above the default, once to a device
template <typename K>
int allow_smem(const Handle* h, K* kernel, size_t smem, bool (&done)[64]) {
  const bool known = h->device >= 0 && h->device < 64;
  if (known && done[h->device]) return MG_OK;
  MG_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  if (known) done[h->device] = true;
  return MG_OK;
}

template <int NT, int NG, bool BACK>
int launch_adapter_as(const Handle* h, const AdapterArgs& a, int64_t jobs, int cs, cudaStream_t st) {
  constexpr size_t smem = AdapterCfg<NT, NG>::SMEM;
  static bool done[64];
  if (int rc = allow_smem(h, adapter_kernel<NT, NG, BACK>, smem, done)) return rc;
  MG_CUDA(launch_clusters(adapter_kernel<NT, NG, BACK>, jobs, cs, smem, st, a));
  return MG_OK;
}
template <bool BACK>
int launch_adapter_rank(const Handle* h, const AdapterArgs& a, cudaStream_t st) {
  const int64_t jobs = a.tiles != nullptr ? (static_cast<int64_t>(a.n_rows) + kAdapterTile - 1) / kAdapterTile + a.n_adapters + 1 : a.n_rows;
  // as many blocks to a tile as run at once, were all tiles full
  const int64_t full = a.tiles != nullptr ? (a.n_rows + kAdapterTile - 1) / kAdapterTile : a.n_rows;
  int cs = 8;
  while (cs > 1 && full * cs > (a.rank > 32 ? 1 : 2) * h->sm_count) cs /= 2;
  switch (padded_rank(a.rank)) {
    case 16: return launch_adapter_as<2, 1, BACK>(h, a, jobs, cs, st);
    case 32: return launch_adapter_as<4, 1, BACK>(h, a, jobs, cs, st);
    case 64: return launch_adapter_as<8, 1, BACK>(h, a, jobs, cs, st);
    default: return launch_adapter_as<8, 2, BACK>(h, a, jobs, cs, st);
  }
}
template <int NT, int NG>
int launch_adapter_grad_as(const Handle* h, const AdapterGradArgs& a, int64_t jobs, int cs, cudaStream_t st) {
  constexpr size_t smem = 256 * (NT * NG * 8 + 1) * sizeof(float);
  static bool done[64];
  if (int rc = allow_smem(h, adapter_grad_kernel<NT, NG>, smem, done)) return rc;
  MG_CUDA(launch_clusters(adapter_grad_kernel<NT, NG>, jobs, cs, smem, st, a));
  return MG_OK;
}

}  // namespace

int adapter_padded_rank(int rank) { return padded_rank(rank); }
int64_t adapter_direct_rows() { return kDirectRows; }
size_t adapter_plan_bytes(int64_t rows, int64_t adapters) { return static_cast<size_t>(plan_layout(rows, adapters).words) * 4; }

int launch_adapter_plan(const Handle* h, const int32_t* ids, const int32_t* counts, const int32_t* pad, int64_t rows, int adapters,
                        void* plan, cudaStream_t st) {
  const PlanLayout p = plan_layout(rows, adapters);
  int32_t* w = static_cast<int32_t*>(plan);
  const int n_tiles = static_cast<int>(p.segs / 4), groups = adapters + 1;
  static bool done[2][64];
  constexpr size_t most = (4 * (MG_ADAPTER_MAX + 1) + 1 + kPlanWarps * (MG_ADAPTER_MAX + 1)) * sizeof(int);
  const size_t smem = (4 * groups + 1 + (ids != nullptr ? kPlanWarps * groups : 0)) * sizeof(int);
  if (ids != nullptr) {
    if (int rc = allow_smem(h, adapter_plan_kernel<false>, most, done[0])) return rc;
    adapter_plan_kernel<false><<<1, kPlanWarps * 32, smem, st>>>(ids, nullptr, nullptr, static_cast<int>(rows), adapters, n_tiles,
                                                                reinterpret_cast<int4*>(w), reinterpret_cast<int2*>(w + p.segs), w + p.order);
  } else {
    const unsigned blocks = static_cast<unsigned>(1 + (rows + kPlanWarps * 32 - 1) / (kPlanWarps * 32));
    adapter_plan_kernel<true><<<blocks, kPlanWarps * 32, smem, st>>>(nullptr, counts, pad, static_cast<int>(rows), adapters, n_tiles,
                                                                    reinterpret_cast<int4*>(w), reinterpret_cast<int2*>(w + p.segs), w + p.order);
  }
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

static AdapterArgs adapter_args(const mg_adapters* d, int64_t rows, const int32_t* ids, const void* plan) {
  AdapterArgs a{};
  a.scale = d->d_scale;
  a.factor = d->factor;
  a.rank = d->rank;
  a.n_adapters = d->n_adapters;
  a.n_rows = static_cast<int>(rows);
  if (plan != nullptr) {
    const PlanLayout p = plan_layout(rows, d->n_adapters);
    const int32_t* w = static_cast<const int32_t*>(plan);
    a.tiles = reinterpret_cast<const int4*>(w);
    a.order = w + p.order;
  } else {
    a.ids = ids;
  }
  return a;
}

int launch_adapter_add(const Handle* h, const mg_adapters* d, const void* x, int64_t ldx, const void* y, int64_t ldy, int64_t rows,
                       const int32_t* ids, const void* plan, void* out, int64_t ldo, void* s, cudaStream_t st) {
  AdapterArgs a = adapter_args(d, rows, ids, plan);
  a.x = static_cast<const uint16_t*>(x); a.ldx = ldx; a.K = static_cast<int>(d->cols);
  a.w1 = static_cast<const uint16_t*>(d->d_down); a.g1 = d->down_stride; a.ld1 = d->ld_down;
  a.w2 = static_cast<const uint16_t*>(d->d_up); a.g2 = d->up_stride; a.ld2 = d->ld_up;
  a.y = static_cast<const uint16_t*>(y); a.ldy = ldy;
  a.out = static_cast<uint16_t*>(out); a.ldo = ldo; a.N = static_cast<int>(d->n_out);
  a.s = static_cast<uint16_t*>(s);
  return launch_adapter_rank<false>(h, a, st);
}

int launch_adapter_grad(const Handle* h, const mg_adapters* d, const void* gout, int64_t ldg, const void* x, int64_t ldx, int64_t rows,
                        const void* plan, const void* s, void* gs, void* gx, int64_t ldgx, void* gdown, void* gup, cudaStream_t st) {
  AdapterArgs a = adapter_args(d, rows, nullptr, plan);
  a.x = static_cast<const uint16_t*>(gout); a.ldx = ldg; a.K = static_cast<int>(d->n_out);
  a.w1 = static_cast<const uint16_t*>(d->d_up); a.g1 = d->up_stride; a.ld1 = d->ld_up;
  a.w2 = static_cast<const uint16_t*>(d->d_down); a.g2 = d->down_stride; a.ld2 = d->ld_down;
  a.out = static_cast<uint16_t*>(gx); a.ldo = ldgx; a.N = gx != nullptr ? static_cast<int>(d->cols) : 0;
  a.s = static_cast<uint16_t*>(gs);
  if (gx != nullptr || gdown != nullptr)
    if (int rc = launch_adapter_rank<true>(h, a, st)) return rc;
  if (gdown == nullptr && gup == nullptr) return MG_OK;
  AdapterGradArgs b{};
  b.wide[0] = static_cast<const uint16_t*>(gout); b.ldw[0] = ldg; b.cols[0] = static_cast<int>(d->n_out);
  b.narrow[0] = static_cast<const uint16_t*>(s); b.out[0] = static_cast<uint16_t*>(gup);
  b.wide[1] = static_cast<const uint16_t*>(x); b.ldw[1] = ldx; b.cols[1] = static_cast<int>(d->cols);
  b.narrow[1] = static_cast<const uint16_t*>(gs); b.out[1] = static_cast<uint16_t*>(gdown);
  for (int i = 0; i < 2; ++i) b.blocks[i] = b.out[i] != nullptr ? (b.cols[i] + 255) / 256 : 0;
  b.scale = a.scale;
  b.factor = a.factor;
  b.rank = a.rank;
  b.order = a.order;
  b.segs = reinterpret_cast<const int2*>(static_cast<const int32_t*>(plan) + plan_layout(rows, d->n_adapters).segs);
  const int64_t jobs = static_cast<int64_t>(d->n_adapters) * (b.blocks[0] + b.blocks[1]);
  // rows of an adapter shared among blocks while each has two steps of 64 rows, were all adapters alike
  int cs = 8;
  while (cs > 1 && rows / d->n_adapters < 128 * cs) cs /= 2;
  switch (padded_rank(a.rank)) {
    case 16: return launch_adapter_grad_as<2, 1>(h, b, jobs, cs, st);
    case 32: return launch_adapter_grad_as<4, 1>(h, b, jobs, cs, st);
    case 64: return launch_adapter_grad_as<8, 1>(h, b, jobs, cs, st);
    default: return launch_adapter_grad_as<8, 2>(h, b, jobs, cs, st);
  }
}

}  // namespace mg
