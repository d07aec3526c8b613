// Products of int8 rows and int8 weights: out[token, n] = bf16(sum_k a[token, k] b[n, k] * a_scale[token] * b_scale[n]), grouped by
// expert or one dense matrix, gate and up rows optionally joined by SwiGLU.  The sums are exact in 32 bits.
//
// A block of eight warps holds 128 weight rows (A of the MMA) against BN tokens (B) in registers; both come through a ring of
// 128-byte steps filled by asynchronous copies.  Few tokens: a warp per 16 weight rows, so that a weight is read from shared memory
// once; 128 tokens: 32 rows x 64 tokens per warp.  For SwiGLU a warp's sixteen rows are eight gate rows and the up rows of the same
// outputs, which then meet in one thread.
// What bounds it: with few tokens the weights' bytes (V2-236B layer, 64 tokens, 5.7 TB/s); with many the warp-wide integer MMAs, whose
// pipe runs 60 % of the cycles at one block of 256 tokens per SM (4096 x 4096 x 7168 367 us, 0.65 POP/s; 8192 601 us, 0.80), between
// the filling of the ring at the start of a tile and the last round of tiles; shared memory 31 %.
// It is deliberately of plain parts: warp-wide MMAs, copies counted by the thread that issued them and block barriers, so nothing in
// it waits for another block, another kernel or a flag.  An earlier form on SM pairs (tensor memory, copies by the tensor engine,
// launched by programmatic dependence) was faster for large batches and stalled without end once in some million passes.
#include "tc.cuh"

namespace mg {

namespace {

constexpr int I8_BM = 128, I8_STEP = 128, I8_THREADS = 256;
constexpr int I8_GROUP = 8;       // token tiles that share a weight tile through L2 before the next weight tile

template <int BN>
struct I8Cfg {
  static constexpr int BLOCKS = BN == 256 ? 1 : 2;                        // per SM
  static constexpr int STAGES = BN == 128 ? 3 : BN <= 32 ? 5 : 4;
  static constexpr int STAGE = (I8_BM + BN) * I8_STEP;
  static constexpr int WN = BN == 256 ? 4 : BN == 128 ? 2 : 1, WM = 8 / WN;               // warps over tokens and over weight rows
  static constexpr int MT = I8_BM / (16 * WM), NT = BN / (8 * WN);
  static constexpr int PITCH = 2 * I8_BM + 16;                            // bytes of a token's outputs on their way out
  static constexpr size_t SMEM = static_cast<size_t>(STAGES) * STAGE;
  static_assert(BN * PITCH <= STAGES * STAGE && BLOCKS * (SMEM + 4096) <= 227 * 1024, "shared memory");
};

struct I8Args {
  const uint8_t* a;
  int64_t lda;
  const float* a_scale;
  int64_t a_rows;
  const uint8_t* b;
  int64_t ldb;
  const float* b_scale;
  uint16_t* out;
  int64_t ldo;
  const int32_t* pad_offsets;     // nullptr: one dense matrix
  const int32_t* counts;
  int n_groups, n_per_group, n_tiles, K;
  int wide;                       // rows of out begin on 16 bytes
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_i8(int* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float scaled(int sum, float w, float t) { return __fmul_rn(__fmul_rn(__int2float_rn(sum), t), w); }
__device__ __forceinline__ uint16_t bf16_bits(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

template <bool SWIGLU, int BN>
__global__ void __launch_bounds__(I8_THREADS, I8Cfg<BN>::BLOCKS) gemm_i8_kernel(const I8Args g) {
  using C = I8Cfg<BN>;
  constexpr int OUTS = SWIGLU ? I8_BM / 2 : I8_BM;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_jp[kMaxExperts + 1];           // token tiles of the experts before
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wm = warp % C::WM, wn = warp / C::WM;
  const uint32_t base = smem_u32(smem);
  const bool dense = g.pad_offsets == nullptr;
  auto count_of = [&](int e) -> int64_t { return dense ? g.a_rows : max(g.counts[e], 0); };
  if (warp == 0) {
    constexpr int RUN = kMaxExperts / 32;
    int sum = 0;
    for (int i = 0; i < RUN; ++i)
      if (lane * RUN + i < g.n_groups) sum += static_cast<int>((count_of(lane * RUN + i) + BN - 1) / BN);
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += v;
    }
    int run = inc - sum;
    for (int i = 0; i < RUN; ++i) {
      const int e = lane * RUN + i;
      if (e >= g.n_groups) break;
      s_jp[e] = run;
      run += static_cast<int>((count_of(e) + BN - 1) / BN);
      if (e == g.n_groups - 1) s_jp[g.n_groups] = run;
    }
  }
  __syncthreads();
  const int64_t total = static_cast<int64_t>(s_jp[g.n_groups]) * g.n_tiles;
  const int steps = (g.K + I8_STEP - 1) / I8_STEP;
  const int chunk = tid & 7, row_in = tid >> 3;    // this thread copies 16-byte piece `chunk` of rows row_in, row_in + 32, ...
  constexpr int BR = BN >= 32 ? BN / 32 : 1;

  for (int64_t job = blockIdx.x; job < total; job += gridDim.x) {
    int lo = 0, hi = g.n_groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<int64_t>(s_jp[mid]) * g.n_tiles <= job) lo = mid; else hi = mid;
    }
    const int e = lo, nt = s_jp[e + 1] - s_jp[e];
    const int64_t local = job - static_cast<int64_t>(s_jp[e]) * g.n_tiles;
    const int grp = static_cast<int>(local / (I8_GROUP * g.n_tiles));
    const int rem = static_cast<int>(local - static_cast<int64_t>(grp) * (I8_GROUP * g.n_tiles));
    const int gt = min(I8_GROUP, nt - grp * I8_GROUP);
    const int n = rem / gt;
    const int64_t first = static_cast<int64_t>(grp * I8_GROUP + rem - n * gt) * BN;
    const int64_t row0 = (dense ? 0 : g.pad_offsets[e]) + first;
    int64_t live = min(count_of(e) - first, g.a_rows - row0);
    if (row0 < 0 || live <= 0) continue;           // the same for the whole block
    const int left = static_cast<int>(min(live, static_cast<int64_t>(BN)));
    const int64_t w0 = static_cast<int64_t>(e) * g.n_per_group;
    // row r of the tile -> row of the group's weights; gate/up rows come in blocks of 128 and 128
    auto w_row = [&](int r) {
      return SWIGLU ? (n >> 1) * 256 + ((r >> 3) & 1) * 128 + (n & 1) * 64 + (r >> 4) * 8 + (r & 7) : n * I8_BM + r;
    };
    const uint8_t* wp[4];
    const uint8_t* tp[BR];
    bool w_ok[4], t_ok[BR];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = w_row(row_in + 32 * i);
      w_ok[i] = r < g.n_per_group;
      wp[i] = g.b + (w0 + (w_ok[i] ? r : 0)) * g.ldb + chunk * 16;
    }
#pragma unroll
    for (int i = 0; i < BR; ++i) {
      const int t = row_in + 32 * i;
      t_ok[i] = t < left;
      tp[i] = g.a + (row0 + (t_ok[i] ? t : 0)) * g.lda + chunk * 16;
    }
    auto load = [&](int kt) {
      if (kt < steps) {
        const uint32_t st = base + (kt % C::STAGES) * C::STAGE;
        const int64_t k = static_cast<int64_t>(kt) * I8_STEP;
        const int have = min(max(g.K - kt * I8_STEP - chunk * 16, 0), 16);       // what lies behind a row's end is not read
        const int64_t at = have > 0 ? k : -chunk * 16;                            // an address inside the row for a copy of nothing
        const uint32_t piece = static_cast<uint32_t>((chunk ^ (row_in & 7)) << 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) copy16(st + (row_in + 32 * i) * I8_STEP + piece, wp[i] + at, w_ok[i] ? have : 0);
#pragma unroll
        for (int i = 0; i < BR; ++i)
          if (BN >= 32 || row_in < BN)
            copy16(st + (I8_BM + row_in + 32 * i) * I8_STEP + piece, tp[i] + at, t_ok[i] ? have : 0);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int acc[C::MT][C::NT][4];
#pragma unroll
    for (int m = 0; m < C::MT; ++m)
#pragma unroll
      for (int x = 0; x < C::NT; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][x][i] = 0;
#pragma unroll
    for (int s = 0; s < C::STAGES - 1; ++s) load(s);
    for (int kt = 0; kt < steps; ++kt) {
      asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 2) : "memory");
      __syncthreads();                             // step kt is there for all, and all have left the stage that is filled next
      load(kt + C::STAGES - 1);
      const uint32_t st = base + (kt % C::STAGES) * C::STAGE;
#pragma unroll
      for (int k = 0; k < I8_STEP / 32; ++k) {
        uint32_t fa[C::MT][4];
#pragma unroll
        for (int m = 0; m < C::MT; ++m) {
          // rows 0-7 and 8-15 of bytes 0-15, then both of bytes 16-31
          const int r = (wm * C::MT + m) * 16 + (lane & 15), c = 2 * k + (lane >> 4);
          ldmatrix4(st + r * I8_STEP + ((c ^ (r & 7)) << 4), fa[m]);
        }
#pragma unroll
        for (int x = 0; x < C::NT; x += 2) {
          // bytes 0-15 and 16-31 of eight tokens, then of the next eight
          uint32_t fb[4];
          const int r = (wn * C::NT + x) * 8 + (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
          ldmatrix4(st + (I8_BM + r) * I8_STEP + ((c ^ (r & 7)) << 4), fb);
#pragma unroll
          for (int m = 0; m < C::MT; ++m) {
            mma_i8(acc[m][x], fa[m], fb[0], fb[1]);
            mma_i8(acc[m][x + 1], fa[m], fb[2], fb[3]);
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                               // the ring is free: outputs pass through it, a token's side by side
    const int col0 = n * OUTS;
#pragma unroll
    for (int m = 0; m < C::MT; ++m) {
      const int r = (wm * C::MT + m) * 16 + (lane >> 2);
      const int r0 = w_row(r), r1 = w_row(r + 8);
      const float s0 = r0 < g.n_per_group ? g.b_scale[w0 + r0] : 0.f, s1 = r1 < g.n_per_group ? g.b_scale[w0 + r1] : 0.f;
#pragma unroll
      for (int x = 0; x < C::NT; ++x)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int t = (wn * C::NT + x) * 8 + 2 * (lane & 3) + j;
          if (t >= left) continue;
          const float ts = g.a_scale[row0 + t];
          const float u = scaled(acc[m][x][j], s0, ts), v = scaled(acc[m][x][2 + j], s1, ts);
          uint8_t* p = smem + t * C::PITCH;
          if (SWIGLU) {
            *reinterpret_cast<uint16_t*>(p + 2 * ((r >> 4) * 8 + (r & 7))) = bf16_bits(silu_f(u) * v);
          } else {
            *reinterpret_cast<uint16_t*>(p + 2 * r) = bf16_bits(u);
            *reinterpret_cast<uint16_t*>(p + 2 * (r + 8)) = bf16_bits(v);
          }
        }
    }
    __syncthreads();
    const int cols = SWIGLU ? g.n_per_group / 2 : g.n_per_group;
    for (int i = tid; i < left * (OUTS / 8); i += I8_THREADS) {
      const int t = i / (OUTS / 8), c = i % (OUTS / 8) * 8;
      const uint8_t* p = smem + t * C::PITCH + 2 * c;
      uint16_t* dst = g.out + (row0 + t) * g.ldo + col0 + c;
      if (g.wide && col0 + c + 8 <= cols) {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(p);
      } else {
        for (int j = 0; j < 8 && col0 + c + j < cols; ++j) dst[j] = reinterpret_cast<const uint16_t*>(p)[j];
      }
    }
    __syncthreads();                               // the next job's copies overwrite what was just read
  }
}

template <bool SWIGLU, int BN>
int launch(const Handle* h, const I8Args& a, int64_t tiles, cudaStream_t st) {
  using C = I8Cfg<BN>;
  static bool done[64];
  if (!(h->device >= 0 && h->device < 64 && done[h->device])) {
    MG_CUDA(cudaFuncSetAttribute(gemm_i8_kernel<SWIGLU, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::SMEM)));
    if (h->device >= 0 && h->device < 64) done[h->device] = true;
  }
  const int64_t most = static_cast<int64_t>(C::BLOCKS) * h->sm_count, jobs = tiles * a.n_tiles;
  gemm_i8_kernel<SWIGLU, BN><<<static_cast<unsigned>(jobs < most ? jobs : most), I8_THREADS, C::SMEM, st>>>(a);
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

template <int BN>
int launch(const Handle* h, const I8Args& a, int64_t rows, bool swiglu, cudaStream_t st) {
  const int64_t tiles = (rows + BN - 1) / BN + (a.pad_offsets != nullptr ? a.n_groups : 0);
  return swiglu ? launch<true, BN>(h, a, tiles, st) : launch<false, BN>(h, a, tiles, st);
}

}  // namespace

int launch_gemm_i8(const Handle* h, const GemmProblem& p, cudaStream_t st) {
  const bool swiglu = p.epilogue == EPI_SWIGLU_BF16, dense = p.pad_offsets == nullptr;
  MG_REQUIRE(p.scales != nullptr && p.a_scales != nullptr && (swiglu || p.epilogue == EPI_PLAIN_BF16), MG_ERR_CONFIG,
             "int8 GEMM: scales of both sides, and bf16 outputs only");
  MG_REQUIRE(p.n_groups >= 1 && p.n_groups <= kMaxExperts && p.K >= 1 && p.K <= kInt8MaxK && p.lda % 16 == 0 && p.ldb % 16 == 0 &&
             p.lda >= p.K && p.ldb >= p.K && p.ldo % 8 == 0 && (dense || p.n_per_group % 256 == 0) &&
             (!swiglu || p.n_per_group % 256 == 0), MG_ERR_SHAPE, "int8 GEMM: K=%d, N=%d, row strides %lld, %lld and %lld", p.K,
             p.n_per_group, static_cast<long long>(p.lda), static_cast<long long>(p.ldb), static_cast<long long>(p.ldo));
  const int64_t rows = dense ? p.dense_rows : p.a_rows;
  I8Args a{static_cast<const uint8_t*>(p.a), p.lda, p.a_scales, rows, static_cast<const uint8_t*>(p.b), p.ldb, p.scales,
           static_cast<uint16_t*>(p.out), p.ldo, p.pad_offsets, p.counts, p.n_groups, p.n_per_group,
           (p.n_per_group + I8_BM - 1) / I8_BM, p.K, reinterpret_cast<uintptr_t>(p.out) % 16 == 0};
  // Tokens of a tile: what a group has on average, whose rows are padded to whole tiles of 128 and one more; of a dense matrix less
  // while fewer than three quarters of the SMs would have a block.  us, 4096 x 4096, by the mean alone and so: 64 tokens 23.1 and
  // 13.9, 256 52.7 and 24.0, 512 52.8 and 35.8; 256 tokens of 1024 x 8192 98 and 24.5; 1024 tokens in 128 blocks of 256 53.8, in 256
  // of 128 60.6.  256 against 128 tokens at most: 8192 x 4096 x 7168 with its rows 631 and 716, Mixtral layer 8192 tokens 8.6 and 9.0 ms.
  // Tiles of 32 tokens from a mean of 5 on, layer: V2-Lite 64 tokens 138 and 143, V2-236B 201 625 and 631, Mixtral 61 273 and 278.
  const int64_t mean = dense ? rows : (rows - 128ll * p.n_groups) / p.n_groups;
  int bn = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : mean <= 192 ? 128 : 256;
  while (dense && bn > 16 && (rows + bn - 1) / bn * a.n_tiles * 4 < 3ll * h->sm_count) bn /= 2;
  switch (bn) {
    case 16: return launch<16>(h, a, rows, swiglu, st);
    case 32: return launch<32>(h, a, rows, swiglu, st);
    case 64: return launch<64>(h, a, rows, swiglu, st);
    case 128: return launch<128>(h, a, rows, swiglu, st);
    default: return launch<256>(h, a, rows, swiglu, st);
  }
}

}  // namespace mg
