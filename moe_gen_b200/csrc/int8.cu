// 8-bit integer activations: quantisation of rows, and the dense product as the library's callers reach it.  The product
// itself is in gemm_i8.cu, the arithmetic of a row in tc.cuh.
#include "tc.cuh"

namespace mg {

namespace {

constexpr int64_t kWarpRows = 1024;      // fewer rows than this have a block each, and its latency
constexpr int kQuantVecs = 8;            // 16-byte vectors of a row a thread keeps in registers at most
// largest |x| of the block's row as bf16 bits (an infinity or NaN is larger than any number)
__device__ __forceinline__ uint32_t block_amax(uint32_t pairs, uint32_t* s_max) {
  const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, max(pairs & 0xFFFFu, pairs >> 16));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
  uint32_t a = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) a = max(a, s_max[i]);
  return a;
}

// A block per row, or per entry of `list` (rows of the experts' buffers; one outside their list_rows rows is skipped).  Rows of
// whole 16-byte vectors; what a thread holds stays in registers between the maximum and the rounding.  Bound by HBM (3 bytes per
// element): 8192 rows of 7168 in 30 us, 16384 of 14336 in 100.
template <int VECS>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const uint4* x, int64_t ldx, int vecs, const int32_t* list,
                                                            int64_t list_rows, uint2* q, int64_t ldq, float* scale) {
  __shared__ uint32_t s_max[8];
  const int64_t row = list != nullptr ? list[blockIdx.x] : static_cast<int64_t>(blockIdx.x);
  if (row < 0 || row >= list_rows) return;
  const uint4* src = x + row * ldx;
  uint4 keep[VECS];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    keep[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < vecs) keep[i] = src[v];
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) m = amax8(m, keep[i]);
  float s, inv;
  row_scale(block_amax(m, s_max), s, inv);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < vecs) q[row * ldq + v] = quantise8(keep[i], inv);
  }
  if (threadIdx.x == 0) scale[row] = s;
}

// The same with a warp per row, for many rows that its lanes can hold: blocks of 64 threads were bound by their number
// (24576 rows of 1408, us, so and now: 26 and 16).
template <int VECS>
__global__ void __launch_bounds__(256) quantize_short_rows_kernel(const uint4* x, int64_t ldx, int vecs, int64_t n, const int32_t* list,
                                                                  int64_t list_rows, uint2* q, int64_t ldq, float* scale) {
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= n) return;
  const int64_t row = list != nullptr ? list[item] : item;
  if (row < 0 || row >= list_rows) return;
  const uint4* src = x + row * ldx;
  uint4 keep[VECS];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = lane + i * 32;
    keep[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < vecs) keep[i] = src[v];
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) m = amax8(m, keep[i]);
  float s, inv;
  row_scale(__reduce_max_sync(0xFFFFFFFFu, max(m & 0xFFFFu, m >> 16)), s, inv);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = lane + i * 32;
    if (v < vecs) q[row * ldq + v] = quantise8(keep[i], inv);
  }
  if (lane == 0) scale[row] = s;
}

// A product of up to kFewRows rows of x in one launch: every block quantises them into shared memory, and a warp multiplies two
// weight rows at a time by them with four-way dot products.  Few rows leave the tensor cores idle and their tiles few (a
// block for 128 weight rows); here every SM streams a share of the weights.
constexpr int kFewRows = 16, kFewWarps = 16, kFewSmem = 96 * 1024;
// Blocks that run at once on an SM, by their registers: 60 to 64 a thread for up to four rows, 108 and 128 for eight and sixteen.  Asked
// of the compiler as a launch bound, it spills: 2 rows 16384x4096 8.6 us without, 10.1 with it.
constexpr int few_blocks(int m) { return m <= 4 ? 2 : 1; }
template <int M>
__global__ void __launch_bounds__(kFewWarps * 32) int8_few_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx, int rows, int cols,
                                                                       const uint8_t* __restrict__ w, int64_t ldw,
                                                                       const float* __restrict__ w_scale, int n_out,
                                                                       __nv_bfloat16* __restrict__ out, int64_t ldo, bool wide) {
  extern __shared__ __align__(16) uint8_t s_q[];           // [M][chunks of 16 bytes], zeros behind the last element
  __shared__ uint32_t s_max[kFewWarps];
  __shared__ float s_scale[M];
  constexpr int ROW_WARPS = kFewWarps / M, STEP = ROW_WARPS * 32, KEEP = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = (cols + 15) >> 4;
  int n0 = (blockIdx.x * kFewWarps + warp) * 2;
  // this warp's first weights on their way while x is quantised
  if (n0 < n_out) {
    const uint8_t* p = w + static_cast<int64_t>(min(n0 + (lane & 1), n_out - 1)) * ldw;
    for (int c = (lane >> 1) * 128; c < cols; c += 16 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + c));
  }
  {
    const int r = warp / ROW_WARPS, t = threadIdx.x - r * STEP;          // ROW_WARPS warps to a row
    const bool live = r < rows;
    const uint16_t* src = x + (live ? r : 0) * ldx;
    const uint4* v4 = reinterpret_cast<const uint4*>(src);
    const int vecs = wide && live ? cols >> 3 : 0;
    uint4 keep[KEEP];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      keep[i] = make_uint4(0u, 0u, 0u, 0u);
      if (t + i * STEP < vecs) keep[i] = __ldg(v4 + t + i * STEP);
    }
#pragma unroll
    for (int i = 0; i < KEEP; ++i) m = amax8(m, keep[i]);
    for (int c = t + KEEP * STEP; c < vecs; c += STEP) m = amax8(m, __ldg(v4 + c));
    m = max(m & 0xFFFFu, m >> 16);
    if (!wide && live)
      for (int c = t; c < cols; c += STEP) m = max(m, __ldg(src + c) & 0x7FFFu);
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if (lane == 0) s_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROW_WARPS; ++i) m = max(m, s_max[r * ROW_WARPS + i]);
    float scale, inv;
    row_scale(m, scale, inv);
    if (t == 0) s_scale[r] = scale;
    uint8_t* q = s_q + static_cast<size_t>(r) * chunks * 16;
    if (wide) {
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (t + i * STEP < chunks * 2) reinterpret_cast<uint2*>(q)[t + i * STEP] = quantise8(keep[i], inv);      // zeros behind the row
      for (int c = t + KEEP * STEP; c < chunks * 2; c += STEP)
        reinterpret_cast<uint2*>(q)[c] = c < vecs ? quantise8(__ldg(v4 + c), inv) : make_uint2(0u, 0u);
    } else {
      for (int c = t; c < chunks * 16; c += STEP) {
        uint32_t lo = 0u, hi;
        if (live && c < cols && inv != 0.f) quantise2(__ldg(src + c), inv, lo, hi);
        q[c] = static_cast<uint8_t>(lo);
      }
    }
  }
  __syncthreads();
  for (; n0 < n_out; n0 += gridDim.x * kFewWarps * 2) {
    const bool two = n0 + 1 < n_out;
    const uint8_t* w0 = w + static_cast<int64_t>(n0) * ldw;
    const uint8_t* w1 = w0 + (two ? ldw : 0);
    int acc0[M], acc1[M];
#pragma unroll
    for (int r = 0; r < M; ++r) acc0[r] = acc1[r] = 0;
    auto dot = [&](int c, const uint4& a, const uint4& b) {
#pragma unroll
      for (int r = 0; r < M; ++r) {
        const uint4 q = *reinterpret_cast<const uint4*>(s_q + (static_cast<size_t>(r) * chunks + c) * 16);
        acc0[r] = __dp4a(static_cast<int>(a.x), static_cast<int>(q.x), acc0[r]);
        acc0[r] = __dp4a(static_cast<int>(a.y), static_cast<int>(q.y), acc0[r]);
        acc0[r] = __dp4a(static_cast<int>(a.z), static_cast<int>(q.z), acc0[r]);
        acc0[r] = __dp4a(static_cast<int>(a.w), static_cast<int>(q.w), acc0[r]);
        acc1[r] = __dp4a(static_cast<int>(b.x), static_cast<int>(q.x), acc1[r]);
        acc1[r] = __dp4a(static_cast<int>(b.y), static_cast<int>(q.y), acc1[r]);
        acc1[r] = __dp4a(static_cast<int>(b.z), static_cast<int>(q.z), acc1[r]);
        acc1[r] = __dp4a(static_cast<int>(b.w), static_cast<int>(q.w), acc1[r]);
      }
    };
    const int whole = cols >> 4;
    int c = lane;
    for (; c + 96 < whole; c += 128) {
      uint4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = __ldg(reinterpret_cast<const uint4*>(w0) + c + 32 * i);
        b[i] = __ldg(reinterpret_cast<const uint4*>(w1) + c + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) dot(c + 32 * i, a[i], b[i]);
    }
    for (; c < whole; c += 32) dot(c, __ldg(reinterpret_cast<const uint4*>(w0) + c), __ldg(reinterpret_cast<const uint4*>(w1) + c));
    if (c == whole && whole < chunks) {                      // the bytes behind the last whole chunk, one by one
      uint32_t a[4] = {0u, 0u, 0u, 0u}, b[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (whole * 16 + i < cols) {
          a[i >> 2] |= static_cast<uint32_t>(w0[whole * 16 + i]) << (8 * (i & 3));
          b[i >> 2] |= static_cast<uint32_t>(w1[whole * 16 + i]) << (8 * (i & 3));
        }
      }
      dot(whole, make_uint4(a[0], a[1], a[2], a[3]), make_uint4(b[0], b[1], b[2], b[3]));
    }
    const float s0 = w_scale[n0], s1 = two ? w_scale[n0 + 1] : 0.f;
#pragma unroll
    for (int r = 0; r < M; ++r) {
      const int a = __reduce_add_sync(0xFFFFFFFFu, acc0[r]), b = __reduce_add_sync(0xFFFFFFFFu, acc1[r]);
      if (lane == 0 && r < rows) {
        out[r * ldo + n0] = __float2bfloat16_rn(__fmul_rn(__fmul_rn(__int2float_rn(a), s_scale[r]), s0));
        if (two) out[r * ldo + n0 + 1] = __float2bfloat16_rn(__fmul_rn(__fmul_rn(__int2float_rn(b), s_scale[r]), s1));
      }
    }
  }
}

// Rows (or listed rows) of any length, alignment and stride, element by element, read twice.
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const uint16_t* x, int64_t ldx, int cols, const int32_t* list,
                                                                int64_t list_rows, uint8_t* q, int64_t ldq, float* scale) {
  __shared__ uint32_t s_max[8];
  const int64_t row = list != nullptr ? list[blockIdx.x] : static_cast<int64_t>(blockIdx.x);
  if (row < 0 || row >= list_rows) return;
  const uint16_t* src = x + row * ldx;
  uint32_t m = 0;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) m = max(m, src[c] & 0x7FFFu);
  float s, inv;
  row_scale(block_amax(m, s_max), s, inv);
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    uint32_t lo, hi;
    quantise2(src[c], inv, lo, hi);
    q[row * ldq + c] = inv == 0.0f ? 0 : static_cast<uint8_t>(lo);
  }
  if (threadIdx.x == 0) scale[row] = s;
}

}  // namespace

// ldx in elements, ldq in bytes; list: nullptr, or the n rows to quantise of list_rows
int launch_quantize_rows(const void* x, int64_t n, int64_t cols, int64_t ldx, void* q, int64_t ldq, float* scale,
                         cudaStream_t st, const int32_t* list, int64_t list_rows) {
  if (n == 0) return MG_OK;
  MG_REQUIRE(n < (1ll << 31), MG_ERR_LIMIT, "quantise: %lld rows", static_cast<long long>(n));
  const int64_t vecs = cols / 8, bound = list == nullptr ? n : list_rows;
  const bool wide = cols % 8 == 0 && ldx % 8 == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(q) % 8 == 0 && vecs <= 256 * kQuantVecs;
  if (wide) {
    // four vectors to a thread, so that short rows do not leave most of a block idle
    int threads = static_cast<int>((vecs + 127) / 128) * 32;
    if (threads > 256) threads = 256;
    if (vecs <= 32 * kQuantVecs && n >= kWarpRows) {
#define MG_QUANT(V)                                                                                                          \
  quantize_short_rows_kernel<V><<<static_cast<unsigned>((n + 7) / 8), 256, 0, st>>>(                                         \
      static_cast<const uint4*>(x), ldx / 8, static_cast<int>(vecs), n, list, bound, static_cast<uint2*>(q), ldq / 8, scale)
      if (vecs <= 128) MG_QUANT(4); else MG_QUANT(kQuantVecs);
      MG_CUDA(cudaGetLastError());
      return MG_OK;
    }
#undef MG_QUANT
#define MG_QUANT(V)                                                                                                          \
  quantize_rows_kernel<V><<<static_cast<unsigned>(n), threads, 0, st>>>(static_cast<const uint4*>(x), ldx / 8,               \
                                                                        static_cast<int>(vecs), list, bound, static_cast<uint2*>(q), \
                                                                        ldq / 8, scale)
    if (vecs <= 4 * threads) MG_QUANT(4); else MG_QUANT(kQuantVecs);
#undef MG_QUANT
    MG_CUDA(cudaGetLastError());
    return MG_OK;
  }
  quantize_rows_any_kernel<<<static_cast<unsigned>(n), 256, 0, st>>>(static_cast<const uint16_t*>(x), ldx, static_cast<int>(cols), list,
                                                                     bound, static_cast<uint8_t*>(q), ldq, scale);
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

// us with x and weights in L2, in a graph, one launch, and two (quantised, then by gemm_i8.cu): 1 row 4096x4096 4.0 and 14.8,
// 8192x8192 8.7 and 25.7; 4 rows 8192x8192 13.8 and 25.3; 8 rows 1024x1024 4.6 and 6.7, 4096x4096 8.3 and 14.5, 8192x2048 (outputs x
// inputs) 8.3 and 9.4, 16384x1024 10.9 and 7.0; 16 rows 512x512 5.5 and 5.4, 1024x2048 8.6 and 9.2, 4096x2048 8.7 and 9.5, 8192x1024
// 10.4 and 7.0 (a warp quantises a row by itself, and every weight meets all rows from shared memory).  A launch takes 3 to 4 us of
// the call's host side, which bounds a call that waits for nothing.
// So beyond four rows up to 2^24 weights, beyond eight up to 2^23 and 2048 inputs.  Never beyond 2^30 outputs, which the kernel
// counts in 32 bits, a whole grid's step past the last one included.
bool int8_in_one_launch(int64_t rows, int64_t n_out, int64_t cols) {
  int m = 1;
  while (m < rows && m < kFewRows) m *= 2;
  if (rows < 1 || rows > kFewRows || m * round_up(cols, 16) > kFewSmem || n_out > 1 << 30) return false;
  return rows <= 4 || (rows <= 8 ? n_out <= (1 << 24) / cols : cols <= 2048 && n_out <= (1 << 23) / cols);
}
template <int M>
static int launch_few(const Handle* h, const void* x, int64_t ldx, int64_t rows, const void* wq, int64_t ldw, const float* w_scale,
                      int64_t n_out, int64_t cols, void* out, int64_t ldo, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(M * round_up(cols, 16));
  static bool done[64];       // asked for whatever this call's rows take: what the kernel declares by itself counts against the default
  if (!(h->device >= 0 && h->device < 64 && done[h->device])) {
    MG_CUDA(cudaFuncSetAttribute(int8_few_rows_kernel<M>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem));
    if (h->device >= 0 && h->device < 64) done[h->device] = true;
  }
  const bool wide = cols % 8 == 0 && ldx % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  // no more blocks than run at once, since each quantises all of x: us, up to three blocks per SM and so, 8 rows 8192x2048 10.2 and
  // 8.3, 2 rows 16384x4096 (outputs x inputs) 10.8 and 8.6, 16 rows 8192x1024 12.1 and 10.4; level where the outputs are few
  const int64_t want = (n_out + 2 * kFewWarps - 1) / (2 * kFewWarps), most = static_cast<int64_t>(h->sm_count) * few_blocks(M);
  int8_few_rows_kernel<M><<<static_cast<unsigned>(want < most ? want : most), kFewWarps * 32, smem, st>>>(
      static_cast<const uint16_t*>(x), ldx, static_cast<int>(rows), static_cast<int>(cols), static_cast<const uint8_t*>(wq), ldw,
      w_scale, static_cast<int>(n_out), static_cast<__nv_bfloat16*>(out), ldo, wide);
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

int launch_int8_few(const Handle* h, const void* x, int64_t ldx, int64_t rows, const void* wq, int64_t ldw, const float* w_scale,
                    int64_t n_out, int64_t cols, void* out, int64_t ldo, cudaStream_t st) {
  if (rows == 1) return launch_few<1>(h, x, ldx, rows, wq, ldw, w_scale, n_out, cols, out, ldo, st);
  if (rows == 2) return launch_few<2>(h, x, ldx, rows, wq, ldw, w_scale, n_out, cols, out, ldo, st);
  if (rows <= 4) return launch_few<4>(h, x, ldx, rows, wq, ldw, w_scale, n_out, cols, out, ldo, st);
  if (rows <= 8) return launch_few<8>(h, x, ldx, rows, wq, ldw, w_scale, n_out, cols, out, ldo, st);
  return launch_few<16>(h, x, ldx, rows, wq, ldw, w_scale, n_out, cols, out, ldo, st);
}

int launch_int8_matmul(const Handle* h, const void* xq, int64_t ldx, const float* x_scale, int64_t rows, const void* wq, int64_t ldw,
                       const float* w_scale, int64_t n_out, int64_t cols, void* out, int64_t ldo, int epilogue, cudaStream_t st) {
  GemmProblem p{};
  p.a = xq; p.a_rows = rows; p.dense_rows = rows; p.lda = ldx; p.a_scales = x_scale;
  p.b = wq; p.ldb = ldw; p.b_i8 = true; p.scales = w_scale; p.n_groups = 1; p.n_per_group = static_cast<int>(n_out);
  p.K = static_cast<int>(cols); p.out = out; p.ldo = ldo; p.epilogue = epilogue;
  return launch_grouped_gemm(h, p, st);
}

}  // namespace mg
