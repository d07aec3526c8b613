// 8-bit integer activations: quantisation of rows, and the dense product as the library's callers reach it.  The product
// itself is the weight-lane GEMM (gemm_wl.cu).
//
// A row x is held as integers q in [-127, 127] and one scale: m = max(max|x|, 2^-100), scale = m / 127, inv = 127 / m (fp32,
// correctly rounded quotients), q = the integer nearest to x * inv, ties to even.  The product is rounded once: the fused
// multiply-add with 1.5 * 2^23 leaves the integer of the exact product in its low bits.  2^-100 keeps inv finite; rows below
// it, rows of zeros among them, come out as zeros.  A row that holds an infinity or a NaN has scale NaN and q = 0, so that
// every product of the row is NaN.
#include "common.cuh"

namespace mg {

namespace {

constexpr int kQuantVecs = 8;            // 16-byte vectors of a row a thread keeps in registers
constexpr float kQuantFloor = 7.888609052210118e-31f;       // 2^-100

__device__ __forceinline__ void row_scale(uint32_t amax_bits, float& scale, float& inv) {
  const float m = fmaxf(__uint_as_float(amax_bits << 16), kQuantFloor);
  const bool finite = amax_bits < 0x7F80u;
  scale = finite ? __fdiv_rn(m, 127.0f) : __int_as_float(0x7FC00000);
  inv = finite ? __fdiv_rn(127.0f, m) : 0.0f;
}
// the two bf16 of a word -> their integers in the low bytes of lo and hi
__device__ __forceinline__ void quantise2(uint32_t pair, float inv, uint32_t& lo, uint32_t& hi) {
  lo = __float_as_uint(__fmaf_rn(__uint_as_float(pair << 16), inv, 12582912.0f));
  hi = __float_as_uint(__fmaf_rn(__uint_as_float(pair & 0xFFFF0000u), inv, 12582912.0f));
}
__device__ __forceinline__ uint32_t quantise4(uint32_t a, uint32_t b, float inv) {
  uint32_t q[4];
  quantise2(a, inv, q[0], q[1]);
  quantise2(b, inv, q[2], q[3]);
  return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}
// largest |x| of the block's row as bf16 bits (an infinity or NaN is larger than any number)
__device__ __forceinline__ uint32_t block_amax(uint32_t pairs, uint32_t* s_max) {
  const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, max(pairs & 0xFFFFu, pairs >> 16));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
  uint32_t a = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) a = max(a, s_max[i]);
  return a;
}

// A block per row, or per entry of `list` (rows of the experts' buffers; a negative one is skipped).  Rows of whole 16-byte
// vectors; what a thread holds stays in registers between the maximum and the rounding.
__global__ void __launch_bounds__(256) quantize_rows_kernel(const uint4* x, int64_t ldx, int vecs, const int32_t* list,
                                                            uint2* q, int64_t ldq, float* scale) {
  chain_wait();
  chain_go();
  __shared__ uint32_t s_max[8];
  const int64_t row = list != nullptr ? list[blockIdx.x] : static_cast<int64_t>(blockIdx.x);
  if (row < 0) return;
  const uint4* src = x + row * ldx;
  uint4 keep[kQuantVecs];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kQuantVecs; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    keep[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < vecs) keep[i] = src[v];
  }
#pragma unroll
  for (int i = 0; i < kQuantVecs; ++i)
    m = __vmaxu2(__vmaxu2(m, keep[i].x & 0x7FFF7FFFu), __vmaxu2(keep[i].y & 0x7FFF7FFFu,
                 __vmaxu2(keep[i].z & 0x7FFF7FFFu, keep[i].w & 0x7FFF7FFFu)));
  float s, inv;
  row_scale(block_amax(m, s_max), s, inv);
  const bool dead = inv == 0.0f;
#pragma unroll
  for (int i = 0; i < kQuantVecs; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < vecs)
      q[row * ldq + v] = dead ? make_uint2(0u, 0u)
                              : make_uint2(quantise4(keep[i].x, keep[i].y, inv), quantise4(keep[i].z, keep[i].w, inv));
  }
  if (threadIdx.x == 0) scale[row] = s;
}

// Rows of any length, alignment and stride, element by element, read twice.
__global__ void __launch_bounds__(256) quantize_rows_any_kernel(const uint16_t* x, int64_t ldx, int cols, uint8_t* q, int64_t ldq,
                                                                float* scale) {
  chain_wait();
  chain_go();
  __shared__ uint32_t s_max[8];
  const int64_t row = blockIdx.x;
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

// ldx in elements, ldq in bytes; list: nullptr, or the n rows to quantise (cols a multiple of 8 then)
int launch_quantize_rows(const Handle* h, const void* x, int64_t n, int64_t cols, int64_t ldx, const int32_t* list, void* q,
                         int64_t ldq, float* scale, cudaStream_t st) {
  if (n == 0) return MG_OK;
  MG_REQUIRE(n < (1ll << 31), MG_ERR_LIMIT, "quantise: %lld rows", static_cast<long long>(n));
  const int64_t vecs = cols / 8;
  const bool wide = cols % 8 == 0 && ldx % 8 == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(q) % 8 == 0 && vecs <= 256 * kQuantVecs;
  if (wide) {
    // four vectors to a thread, so that short rows do not leave most of a block idle
    int threads = static_cast<int>((vecs + 127) / 128) * 32;
    if (threads > 256) threads = 256;
    MG_CUDA(launch_chained(h, quantize_rows_kernel, static_cast<unsigned>(n), threads, 0, st, static_cast<const uint4*>(x),
                           ldx / 8, static_cast<int>(vecs), list, static_cast<uint2*>(q), ldq / 8, scale));
    return MG_OK;
  }
  MG_REQUIRE(list == nullptr, MG_ERR_SHAPE, "quantise: listed rows of %lld elements", static_cast<long long>(cols));
  MG_CUDA(launch_chained(h, quantize_rows_any_kernel, static_cast<unsigned>(n), 256, 0, st, static_cast<const uint16_t*>(x), ldx,
                         static_cast<int>(cols), static_cast<uint8_t*>(q), ldq, scale));
  return MG_OK;
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
