// The residual's addition and the RMS norm behind it in one pass, rows out in bf16 or in 8-bit integers, and the gradient.
//   h = bf16(x + residual), rstd = 1 / sqrt(mean(h^2) + eps), v = w * (h * rstd) in fp32, y = bf16(v)
//   8 bits: m = max(max|v|, 2^-100), scale = m / 127, q = v * (127 / m) to the nearest, ties to even
// h is rounded because it is stored so, and the norm is of what is stored; v is rounded once.  In front of the block
// y = bf16(w * bf16(h * rstd)), mg_rmsnorm's bits, whose module the block's parity is with.
#include "tc.cuh"

namespace mg {

namespace {

constexpr int kNormLanes = 256;          // lanes over which a row's squares are summed, whatever the kernel (as in rmsnorm_kernel)
// From this many rows of at most 1024 columns on a warp takes a row; us, a warp to a row and a block to a row, bf16 rows (8-bit rows):
//   512 columns: 1024 rows 2.6 (2.8) and 2.5 (3.3), 2048 rows 2.8 (3.1) and 3.6 (5.1), 16384 rows 10.1 (11.0) and 20.7 (29.5)
//   1024 columns: 1024 rows 3.4 (3.7) and 2.7 (3.4), 2048 rows 3.8 (4.2) and 4.1 (5.3), 16384 rows 21.4 (21.3) and 26.7 (33.6)
//   2048 columns: 2048 rows 7.4 (8.6) and 6.0 (7.0), 8192 rows 25.1 (26.1) and 21.5 (22.6): the block, at any number of rows
constexpr int64_t kNormWarpRows = 2048;

enum NormOut { NORM_BF16, NORM_AS_MODULE, NORM_INT8 };
struct NormArgs {
  const uint16_t* x;
  int64_t ldx;
  const uint16_t* res;       // nullptr: h = x
  int64_t ldr;
  const uint16_t* w;
  float eps;
  int64_t n;
  int cols;
  uint16_t* sum;             // h, where there is a residual
  int64_t lds;
  void* out;                 // bf16 rows, or bytes with their scales
  int64_t ldo;
  float* scale;
};

__device__ __forceinline__ uint4 add8(const uint4& a, const uint4& b) {
  float f[8], g[8];
  unpack8(a, f);
  unpack8(b, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __fadd_rn(f[i], g[i]);
  return pack8(f);
}
__device__ __forceinline__ float squares8(const uint4& q, float sum) {
  float f[8];
  unpack8(q, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = fmaf(f[i], f[i], sum);
  return sum;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
__device__ __forceinline__ float rstd_of(float sum, int cols, float eps) { return 1.0f / sqrtf(sum / static_cast<float>(cols) + eps); }
template <int OUT>
__device__ __forceinline__ float normal(float h, float w, float rstd) {
  const float n = __fmul_rn(h, rstd);
  return __fmul_rn(w, OUT == NORM_AS_MODULE ? round_bf16(n) : n);
}
template <int OUT>
__device__ __forceinline__ uint4 rounded8(const uint4& h, const uint4& w, float rstd) {
  float f[8], g[8];
  unpack8(h, f);
  unpack8(w, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = normal<OUT>(f[i], g[i], rstd);
  return pack8(f);
}
__device__ __forceinline__ void normal8(const uint4& h, const uint4& w, float rstd, float* f) {
  float g[8];
  unpack8(h, f);
  unpack8(w, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = normal<NORM_INT8>(f[i], g[i], rstd);
}
// |v| as bits, which order as the numbers do; infinities and NaN are larger than any number
__device__ __forceinline__ uint32_t amax_bits8(uint32_t m, const float* f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  return m;
}
__device__ __forceinline__ void row_scale_f32(uint32_t amax, float& scale, float& inv) {
  const float m = fmaxf(__uint_as_float(amax), kQuantFloor);
  const bool finite = amax < 0x7F800000u;
  scale = finite ? __fdiv_rn(m, 127.0f) : __int_as_float(0x7FC00000);
  inv = finite ? __fdiv_rn(127.0f, m) : 0.0f;
}
__device__ __forceinline__ uint32_t byte_of(float v, float inv) { return __float_as_uint(__fmaf_rn(v, inv, 12582912.0f)); }
__device__ __forceinline__ uint2 bytes8(const float* f, float inv) {
  if (inv == 0.0f) return make_uint2(0u, 0u);
  uint32_t q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = byte_of(f[i], inv);
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
  return make_uint2(w[0], w[1]);
}

// A block per row of whole 16-byte vectors, which stay in registers between the sum and the output: each byte is moved once, and
// memory is what bounds it.  16384 rows of 7168 columns with a residual (four rows' bytes moved per row): 136.5 us, 6.9 TB/s; 8-bit
// rows, 8192 of them: 66.7 us, 6.2 TB/s; one row of 2048 columns: 1.8 us, a launch and one trip to memory.
template <int VECS, int OUT>
__global__ void __launch_bounds__(kNormLanes) add_norm_kernel(const NormArgs a) {
  __shared__ float s_sum[kNormLanes / 32];
  __shared__ uint32_t s_max[kNormLanes / 32];
  const int64_t row = blockIdx.x;
  const int vecs = a.cols >> 3, warp = threadIdx.x >> 5;
  const uint4* x = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
  const uint4* w = reinterpret_cast<const uint4*>(a.w);
  uint4 keep[VECS], wk[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = threadIdx.x + i * kNormLanes;
    keep[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < vecs) keep[i] = x[v];
  }
  if (a.res != nullptr) {
    const uint4* r = reinterpret_cast<const uint4*>(a.res + row * a.ldr);
    uint4* h = reinterpret_cast<uint4*>(a.sum + row * a.lds);
    uint4 other[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = threadIdx.x + i * kNormLanes;
      if (v < vecs) other[i] = r[v];
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = threadIdx.x + i * kNormLanes;
      if (v < vecs) h[v] = keep[i] = add8(keep[i], other[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = threadIdx.x + i * kNormLanes;
    wk[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < vecs) wk[i] = w[v];
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) sum = squares8(keep[i], sum);
  sum = warp_sum(sum);
  if ((threadIdx.x & 31) == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < kNormLanes / 32; ++i) sum += s_sum[i];
  const float rstd = rstd_of(sum, a.cols, a.eps);
  if (OUT != NORM_INT8) {
    uint4* y = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.ldo);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = threadIdx.x + i * kNormLanes;
      if (v < vecs) y[v] = rounded8<OUT>(keep[i], wk[i], rstd);
    }
    return;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    float f[8];
    normal8(keep[i], wk[i], rstd, f);
    m = amax_bits8(m, f);
  }
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if ((threadIdx.x & 31) == 0) s_max[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kNormLanes / 32; ++i) m = max(m, s_max[i]);
  float scale, inv;
  row_scale_f32(m, scale, inv);
  uint2* q = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.out) + row * a.ldo);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = threadIdx.x + i * kNormLanes;
    float f[8];
    normal8(keep[i], wk[i], rstd, f);
    if (v < vecs) q[v] = bytes8(f, inv);
  }
  if (threadIdx.x == 0) a.scale[row] = scale;
}

// A warp per row, for many short rows, where a block's start and its meeting cost more than its bytes.  Its lanes hold what lanes 32
// apart would hold in a block, summed in the same order.
template <int VECS, int OUT>
__global__ void __launch_bounds__(256) add_norm_short_kernel(const NormArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= a.n) return;
  const int vecs = a.cols >> 3;
  const uint4* x = reinterpret_cast<const uint4*>(a.x + row * a.ldx);
  const uint4* w = reinterpret_cast<const uint4*>(a.w);
  uint4 keep[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = lane + i * 32;
    keep[i] = make_uint4(0u, 0u, 0u, 0u);
    if (v < vecs) keep[i] = x[v];
  }
  if (a.res != nullptr) {
    const uint4* r = reinterpret_cast<const uint4*>(a.res + row * a.ldr);
    uint4* h = reinterpret_cast<uint4*>(a.sum + row * a.lds);
    uint4 other[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = lane + i * 32;
      if (v < vecs) other[i] = r[v];
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = lane + i * 32;
      if (v < vecs) h[v] = keep[i] = add8(keep[i], other[i]);
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < VECS; ++i) sum += warp_sum(squares8(keep[i], 0.f));
  const float rstd = rstd_of(sum, a.cols, a.eps);
  if (OUT != NORM_INT8) {
    uint4* y = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.ldo);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = lane + i * 32;
      if (v < vecs) y[v] = rounded8<OUT>(keep[i], __ldg(w + v), rstd);
    }
    return;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = lane + i * 32;
    float f[8];
    if (v < vecs) {
      normal8(keep[i], __ldg(w + v), rstd, f);
      m = amax_bits8(m, f);
    }
  }
  float scale, inv;
  row_scale_f32(__reduce_max_sync(0xFFFFFFFFu, m), scale, inv);
  uint2* q = reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.out) + row * a.ldo);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = lane + i * 32;
    float f[8];
    if (v < vecs) {
      normal8(keep[i], __ldg(w + v), rstd, f);
      q[v] = bytes8(f, inv);
    }
  }
  if (lane == 0) a.scale[row] = scale;
}

// Rows of any length, alignment and stride, element by element.  What is not kept is read again: h, where it was written, by
// the thread that wrote it, so that x or the residual may be where it goes.  8192 rows of 7001 columns with a residual: 322 us, 1.4 TB/s, 8-bit
// rows 269 (7168 columns in vectors: 70 and 67); 7168 columns 7173 apart 329 and 274.  Bound by its loads, of two bytes each and 16 apart in a
// warp, and by reading h three times.
template <int OUT>
__global__ void __launch_bounds__(kNormLanes) add_norm_any_kernel(const NormArgs a) {
  __shared__ float s_sum[kNormLanes / 32];
  __shared__ uint32_t s_max[kNormLanes / 32];
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5;
  const uint16_t* x = a.x + row * a.ldx;
  auto f32 = [](uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); };
  float sum = 0.f;
  for (int64_t v = threadIdx.x; v * 8 < a.cols; v += kNormLanes)
    for (int c = static_cast<int>(v) * 8; c < a.cols && c < static_cast<int>(v) * 8 + 8; ++c) {
      float f = f32(x[c]);
      if (a.res != nullptr) {
        const uint16_t b = __bfloat16_as_ushort(__float2bfloat16_rn(__fadd_rn(f, f32(a.res[row * a.ldr + c]))));
        a.sum[row * a.lds + c] = b;
        f = f32(b);
      }
      sum = fmaf(f, f, sum);
    }
  const uint16_t* h = a.res != nullptr ? a.sum + row * a.lds : x;
  sum = warp_sum(sum);
  if ((threadIdx.x & 31) == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.f;
  for (int i = 0; i < kNormLanes / 32; ++i) sum += s_sum[i];
  const float rstd = rstd_of(sum, a.cols, a.eps);
  uint32_t m = 0;
  for (int64_t v = threadIdx.x; v * 8 < a.cols; v += kNormLanes)
    for (int c = static_cast<int>(v) * 8; c < a.cols && c < static_cast<int>(v) * 8 + 8; ++c) {
      const float v = normal<OUT>(f32(h[c]), f32(a.w[c]), rstd);
      if (OUT == NORM_INT8)
        m = max(m, __float_as_uint(v) & 0x7FFFFFFFu);
      else
        static_cast<uint16_t*>(a.out)[row * a.ldo + c] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
    }
  if (OUT != NORM_INT8) return;
  m = __reduce_max_sync(0xFFFFFFFFu, m);
  if ((threadIdx.x & 31) == 0) s_max[warp] = m;
  __syncthreads();
  for (int i = 0; i < kNormLanes / 32; ++i) m = max(m, s_max[i]);
  float scale, inv;
  row_scale_f32(m, scale, inv);
  for (int64_t v = threadIdx.x; v * 8 < a.cols; v += kNormLanes)
    for (int c = static_cast<int>(v) * 8; c < a.cols && c < static_cast<int>(v) * 8 + 8; ++c)
      static_cast<uint8_t*>(a.out)[row * a.ldo + c] =
          inv == 0.0f ? 0 : static_cast<uint8_t>(byte_of(normal<OUT>(f32(h[c]), f32(a.w[c]), rstd), inv));
  if (threadIdx.x == 0) a.scale[row] = scale;
}

// ---- gradient ----------------------------------------------------------------------------
// With n = h * rstd (the forward's roundings count as the identity):
//   gx = rstd * (w gy - n mean(w gy n)) + gh,   gw = sum over rows of gy n
// mean(w gy n) = rstd sum(w gy h) / cols, so that both sums of a row come from one reading.  Blocks stay and take rows in turn; a
// thread holds the same columns of every row, and its share of gw in fp32.  The shares are summed by a second launch, in the order of
// the blocks, or, few rows, in the same one by a cluster's blocks, so that the same rows and columns give the same bits.
// 8192 rows of 7168 columns with gh: 77 us for 470 MB, 6.1 TB/s, where instructions are what it waits for next to memory: two rows meet at
// once, by sums of which a warp's halves take one each (one row to a meeting and ten exchanges to its sums: 86 us), and what no copy fills
// is zeros in the ring, so that nothing is selected (rows of 16384 columns 145 and 115 us).  Loads into registers took 152 us.  Rows off
// 16-byte vectors are loaded so still, by elements and twice: 8192 rows of 7001 columns 276 us, 1.7 TB/s.
struct NormGradArgs {
  const uint16_t* gy;
  int64_t ldgy;
  const uint16_t* h;
  int64_t ldh;
  const uint16_t* w;
  float eps;
  int64_t n;
  int cols;
  const uint16_t* gh;        // nullptr: none
  int64_t ldgh;
  uint16_t* gx;              // nullptr: not wanted
  int64_t ldgx;
  float* parts;              // [shares][cols], nullptr: gw is not wanted, or
  float* gw;                 // summed here, by one cluster
  int lanes;                 // threads to a row
};
constexpr int kGradThreads = 1024, kGradMaxCols = 2 * 8 * kGradThreads;      // up to two vectors of a row to a thread
// rows on their way at once: 48 bytes to a thread, a vector and a row
template <int VECS>
constexpr int kGradStages = VECS == 1 ? 4 : 2;

template <bool WIDE>
__device__ __forceinline__ uint4 load8(const uint16_t* p, int c, int cols) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (WIDE) {
    if (c < cols) v = *reinterpret_cast<const uint4*>(p + c);
  } else {
    uint32_t* u = &v.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) u[i >> 1] |= static_cast<uint32_t>(p[c + i]) << (16 * (i & 1));
  }
  return v;
}

__device__ __forceinline__ void pairs8(const uint4& v, float2* f) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xFFFF0000u));
}
// bytes: 16, or 0 for zeros
__device__ __forceinline__ void copy_vec(uint4* to, const uint16_t* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(bytes) : "memory");
}

__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Sums over a warp of two numbers of each of R rows: the lanes of a 2 R-th of the warp end with one of them, first a[0], then b[0], a[1], b[1].
// Halves of the warp hand each other what they do not go on with, so that there are 5 or 6 exchanges and not 10 R.
template <int R>
__device__ __forceinline__ float warp_sums(const float (&a)[R], const float (&b)[R]) {
  const int lane = threadIdx.x & 31;
  float v;
  if (R == 1) {
    v = lane & 16 ? b[0] : a[0];
    v += __shfl_xor_sync(0xFFFFFFFFu, lane & 16 ? a[0] : b[0], 16);
    v += __shfl_xor_sync(0xFFFFFFFFu, v, 8);
  } else {
    float x = lane & 16 ? a[R - 1] : a[0], y = lane & 16 ? b[R - 1] : b[0];
    x += __shfl_xor_sync(0xFFFFFFFFu, lane & 16 ? a[0] : a[R - 1], 16);
    y += __shfl_xor_sync(0xFFFFFFFFu, lane & 16 ? b[0] : b[R - 1], 16);
    v = lane & 8 ? y : x;
    v += __shfl_xor_sync(0xFFFFFFFFu, lane & 8 ? x : y, 8);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// WIDE: rows of whole 16-byte vectors, several of them on their way to shared memory at a time.  A thread copies what it reads itself, so
// that it waits for its own copies only.
// FEW: the grid is one cluster, which sums the shares too.
template <int VECS, bool WIDE, bool FEW>
__global__ void __launch_bounds__(kGradThreads, 1) norm_grad_kernel(const NormGradArgs a) {
  constexpr int STAGES = kGradStages<VECS>, R = WIDE ? STAGES / 2 : 1;          // R: rows to a turn, which meet once
  extern __shared__ __align__(16) uint4 s_rows[];                // [stage][h, gy, gh][vector][thread]
  __shared__ float s_sum[2][2 * R][kGradThreads / 32];
  const int lanes = a.lanes, sub = threadIdx.x / lanes, t = threadIdx.x - sub * lanes, rows = blockDim.x / lanes;
  const int warp = threadIdx.x >> 5, warps = lanes >> 5;
  const bool with_h = a.gh != nullptr && a.gx != nullptr;
  float2 w[VECS][4], acc[VECS][4];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    pairs8(load8<WIDE>(a.w, (t + i * lanes) * 8, a.cols), w[i]);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.f, 0.f);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * rows, first = static_cast<int64_t>(blockIdx.x) * rows;
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  uint4* mine = s_rows + threadIdx.x;
  auto slot = [&](int stage, int which, int i) { return mine + ((stage * 3 + which) * VECS + i) * blockDim.x; };
  // the next row to fetch, and this thread's columns of it
  int64_t ahead = first + sub;
  const int64_t there = ahead < a.n ? ahead : 0;
  const uint16_t *ph = a.h + there * a.ldh + t * 8, *pg = a.gy + there * a.ldgy + t * 8, *pr = a.gh + there * a.ldgh + t * 8;
  const int64_t sh = step * a.ldh, sg = step * a.ldgy, sr = step * a.ldgh;
  auto fetch = [&](int stage) {
    const int bytes = ahead < a.n ? 16 : 0;                      // rows behind the last: zeros, by the address of one before
#pragma unroll
    for (int i = 0; i < VECS; ++i)
      if ((t + i * lanes) * 8 < a.cols) {
        copy_vec(slot(stage, 0, i), ph + i * lanes * 8, bytes);
        copy_vec(slot(stage, 1, i), pg + i * lanes * 8, bytes);
        if (with_h) copy_vec(slot(stage, 2, i), pr + i * lanes * 8, bytes);
      }
    ahead += step;
    if (ahead < a.n) { ph += sh; pg += sg; pr += sr; }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (WIDE) {                                                    // what no copy fills: columns behind the last, and rows that are not given
    for (int k = 0; k < STAGES; ++k)
#pragma unroll
      for (int i = 0; i < VECS; ++i)
#pragma unroll
        for (int which = 0; which < 3; ++which)
          if ((t + i * lanes) * 8 >= a.cols || (which == 2 && !with_h)) *slot(k, which, i) = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int k = 0; k < STAGES - R; ++k) fetch(k);
  }
  int turn = 0, stage = 0;                                       // of the turn's first row
  for (int64_t base = first; base < a.n; base += R * step, turn ^= 1) {
    if (WIDE) {
#pragma unroll
      for (int j = 0; j < R; ++j) fetch((stage + STAGES - R + j) % STAGES);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - R) : "memory");
    }
    auto take = [&](const uint16_t* from, int64_t ld, int which, int i, int j) {
      if (WIDE) return *slot((stage + j) % STAGES, which, i);
      const int64_t row = base + j * step + sub;
      return load8<false>(from + row * ld, (t + i * lanes) * 8, row < a.n && (which != 2 || with_h) ? a.cols : 0);
    };
    float ss[R], sp[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float2 s2 = make_float2(0.f, 0.f), p2 = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        float2 fh[4], fg[4];
        pairs8(take(a.h, a.ldh, 0, i, j), fh);
        pairs8(take(a.gy, a.ldgy, 1, i, j), fg);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s2 = __ffma2_rn(fh[e], fh[e], s2);
          p2 = __ffma2_rn(__fmul2_rn(w[i][e], fg[e]), fh[e], p2);
        }
      }
      ss[j] = s2.x + s2.y;
      sp[j] = p2.x + p2.y;
    }
    const int lane = threadIdx.x & 31;
    constexpr int EACH = 16 / R;                                 // lanes that end with a sum
    float v = warp_sums<R>(ss, sp);
    if (warps > 1) {
      if (lane % EACH == 0) s_sum[turn][lane / EACH][warp] = v;
      __syncthreads();               // the other half of s_sum is written in the next turn: no thread is two turns ahead
#pragma unroll
      for (int j = 0; j < R; ++j) {
        ss[j] = lane < warps ? s_sum[turn][2 * j][sub * warps + lane] : 0.f;
        sp[j] = lane < warps ? s_sum[turn][2 * j + 1][sub * warps + lane] : 0.f;
      }
      v = warp_sums<R>(ss, sp);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      ss[j] = __shfl_sync(0xFFFFFFFFu, v, 2 * j * EACH);
      sp[j] = __shfl_sync(0xFFFFFFFFu, v, (2 * j + 1) * EACH);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int64_t row = base + j * step + sub;
      const bool live = row < a.n;
      const float rstd = live ? rsqrtf(fmaf(ss[j], inv_cols, a.eps)) : 0.f;
      const float2 r2 = make_float2(rstd, rstd);
      const float c = -rstd * rstd * (sp[j] * inv_cols);
      const float2 c2 = make_float2(c, c);
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        float2 fh[4], fg[4], fr[4];
        pairs8(take(a.h, a.ldh, 0, i, j), fh);
        pairs8(take(a.gy, a.ldgy, 1, i, j), fg);
        pairs8(take(a.gh, a.ldgh, 2, i, j), fr);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[i][e] = __ffma2_rn(fg[e], __fmul2_rn(fh[e], r2), acc[i][e]);
          fr[e] = __ffma2_rn(r2, __ffma2_rn(fh[e], c2, __fmul2_rn(w[i][e], fg[e])), fr[e]);
        }
        if (a.gx == nullptr || !live) continue;
        const int at = (t + i * lanes) * 8;
        uint16_t* dst = a.gx + row * a.ldgx;
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(fr[e].x, fr[e].y);
          u[e] = *reinterpret_cast<const uint32_t*>(&v);
        }
        if (WIDE) {
          if (at < a.cols) *reinterpret_cast<uint4*>(dst + at) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (at + e < a.cols) dst[at + e] = static_cast<uint16_t>(u[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
    stage = (stage + R) % STAGES;
  }
  if (FEW) {
    if (a.gw == nullptr) return;
    float* part = reinterpret_cast<float*>(s_rows);              // [rows][cols], where the ring is
    copies_done();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = (t + i * lanes) * 8 + j;
        if (c < a.cols) part[sub * a.cols + c] = j & 1 ? acc[i][j >> 1].y : acc[i][j >> 1].x;
      }
    cluster_sync_all();
    const int blocks = static_cast<int>(gridDim.x);
    for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < a.cols; c += blocks * blockDim.x) {
      float v = 0.f;
      for (int k = 0; k < blocks; ++k) {
        const uint32_t there = map_to_cta(smem_u32(part + c), k);
        for (int r = 0; r < rows; ++r) v += ld_cluster_f32(there + r * a.cols * 4);
      }
      a.gw[c] = v;
    }
    cluster_sync_all();              // no block leaves while another reads its share
    return;
  }
  if (a.parts == nullptr) return;
  float* part = a.parts + (static_cast<int64_t>(blockIdx.x) * rows + sub) * a.cols;
#pragma unroll
  for (int i = 0; i < VECS; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = (t + i * lanes) * 8 + j;
      if (c < a.cols) part[c] = j & 1 ? acc[i][j >> 1].y : acc[i][j >> 1].x;
    }
}

// gw[c] = the sum of the shares of column c: 32 columns and 32 shares at a time to a block
__global__ void __launch_bounds__(1024) norm_grad_sum_kernel(const float* parts, int shares, int cols, float* gw) {
  __shared__ float s[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, c = blockIdx.x * 32 + x;
  float v = 0.f;
  if (c < cols)
    for (int p = y; p < shares; p += 32) v += parts[static_cast<int64_t>(p) * cols + c];
  s[y][x] = v;
  __syncthreads();
  v = warp_sum(s[x][y]);             // warp y: the 32 sums of column y of the block
  if (x == 0 && blockIdx.x * 32 + y < cols) gw[blockIdx.x * 32 + y] = v;
}

// Two launches and one, us in a graph: 1 row of 2048 columns 4.8 and 5.2, 16 rows 5.0 and 5.3, 37 rows 5.3 and 7.2, 64 rows 6.0 and 8.5,
// 128 rows 5.9 and 12.5.  A call from Python at 37 rows: 18.0 and 12.2, since two launches and their scratch cost the host more than
// the device gains; from MG_NORM_GRAD_FEW rows on the device's side wins.
constexpr int kGradCluster = 8;
struct NormGradPlan { int vecs, lanes, threads, blocks, shares; bool few; };
NormGradPlan norm_grad_plan(const Handle* h, int64_t n, int64_t cols) {
  NormGradPlan p;
  const int vecs = static_cast<int>((cols + 7) / 8);
  p.vecs = vecs <= kGradThreads ? 1 : 2;
  p.lanes = (vecs + 32 * p.vecs - 1) / (32 * p.vecs) * 32;
  p.threads = p.lanes >= 256 ? p.lanes : 256 / p.lanes * p.lanes;
  const int rows = p.threads / p.lanes;
  const int64_t want = (n + rows - 1) / rows, most = static_cast<int64_t>(h->sm_count) * (p.threads > 512 ? 1 : p.threads > 256 ? 2 : 4);
  p.few = n <= MG_NORM_GRAD_FEW;
  p.blocks = p.few ? kGradCluster : static_cast<int>(want < most ? want : most);
  p.shares = p.few ? 0 : p.blocks * rows;
  return p;
}

bool on16(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

template <int OUT>
int launch_add_norm_as(const NormArgs& a, cudaStream_t st) {
  const int vecs = a.cols / 8;
  const bool wide = a.cols % 8 == 0 && on16(a.x, a.ldx) && (a.res == nullptr || (on16(a.res, a.ldr) && on16(a.sum, a.lds))) &&
                    on16(a.w, 0) && vecs <= 8 * kNormLanes && reinterpret_cast<uintptr_t>(a.out) % (OUT == NORM_INT8 ? 8 : 16) == 0 && a.ldo % 8 == 0;
  const unsigned rows = static_cast<unsigned>(a.n), eighth = static_cast<unsigned>((a.n + 7) / 8);
  if (!wide) add_norm_any_kernel<OUT><<<rows, kNormLanes, 0, st>>>(a);
  else if (a.n >= kNormWarpRows && vecs <= 64) add_norm_short_kernel<2, OUT><<<eighth, 256, 0, st>>>(a);
  else if (a.n >= kNormWarpRows && vecs <= 128) add_norm_short_kernel<4, OUT><<<eighth, 256, 0, st>>>(a);
  else if (vecs <= kNormLanes) add_norm_kernel<1, OUT><<<rows, kNormLanes, 0, st>>>(a);
  else if (vecs <= 2 * kNormLanes) add_norm_kernel<2, OUT><<<rows, kNormLanes, 0, st>>>(a);
  else if (vecs <= 4 * kNormLanes) add_norm_kernel<4, OUT><<<rows, kNormLanes, 0, st>>>(a);
  else add_norm_kernel<8, OUT><<<rows, kNormLanes, 0, st>>>(a);
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

template <int VECS, bool WIDE>
int launch_norm_grad_as(const Handle* h, const NormGradArgs& a, const NormGradPlan& p, cudaStream_t st) {
  const size_t ring = WIDE ? static_cast<size_t>(p.threads) * kGradStages<VECS> * 3 * VECS * sizeof(uint4) : 0;
  constexpr size_t most = kGradThreads * kGradStages<VECS> * 3 * VECS * sizeof(uint4);
  if (p.few) {
    const size_t part = static_cast<size_t>(p.threads / p.lanes) * a.cols * sizeof(float);
    static bool done[64];
    if (int rc = allow_smem(h, norm_grad_kernel<VECS, WIDE, true>, most, done)) return rc;
    MG_CUDA(launch_clusters(norm_grad_kernel<VECS, WIDE, true>, 1, p.blocks, p.threads, ring > part ? ring : part, st, a));
    return MG_OK;
  }
  static bool done[64];
  if (int rc = allow_smem(h, norm_grad_kernel<VECS, WIDE, false>, most, done)) return rc;
  norm_grad_kernel<VECS, WIDE, false><<<p.blocks, p.threads, ring, st>>>(a);
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

}  // namespace

// scale: nullptr for bf16 rows, ldo in elements of out either way; as_module: bf16 rows rounded as mg_rmsnorm's
int launch_add_norm(const void* x, int64_t ldx, const void* res, int64_t ldr, const void* w, float eps, int64_t n, int64_t cols,
                    void* sum, int64_t lds, void* out, int64_t ldo, float* scale, bool as_module, cudaStream_t st) {
  if (n == 0) return MG_OK;
  NormArgs a{static_cast<const uint16_t*>(x), ldx, static_cast<const uint16_t*>(res), ldr, static_cast<const uint16_t*>(w), eps, n,
             static_cast<int>(cols), static_cast<uint16_t*>(sum), lds, out, ldo, scale};
  if (scale != nullptr) return launch_add_norm_as<NORM_INT8>(a, st);
  return as_module ? launch_add_norm_as<NORM_AS_MODULE>(a, st) : launch_add_norm_as<NORM_BF16>(a, st);
}

int64_t norm_grad_max_cols() { return kGradMaxCols; }

size_t norm_grad_ws_bytes(const Handle* h, int64_t n, int64_t cols) {
  return static_cast<size_t>(norm_grad_plan(h, n, cols).shares) * cols * sizeof(float);
}

int launch_norm_grad(const Handle* h, const void* gy, int64_t ldgy, const void* hrows, int64_t ldh, const void* w, float eps, int64_t n,
                     int64_t cols, const void* gh, int64_t ldgh, void* gx, int64_t ldgx, float* gw, void* ws, cudaStream_t st) {
  if (n == 0) {
    if (gw != nullptr) MG_CUDA(cudaMemsetAsync(gw, 0, cols * sizeof(float), st));
    return MG_OK;
  }
  const NormGradPlan p = norm_grad_plan(h, n, cols);
  NormGradArgs a{static_cast<const uint16_t*>(gy), ldgy, static_cast<const uint16_t*>(hrows), ldh, static_cast<const uint16_t*>(w), eps, n,
                 static_cast<int>(cols), static_cast<const uint16_t*>(gh), ldgh, static_cast<uint16_t*>(gx), ldgx,
                 gw != nullptr && !p.few ? static_cast<float*>(ws) : nullptr, p.few ? gw : nullptr, p.lanes};
  const bool wide = cols % 8 == 0 && on16(gy, ldgy) && on16(hrows, ldh) && on16(w, 0) && (gh == nullptr || on16(gh, ldgh)) &&
                    (gx == nullptr || on16(gx, ldgx));
  const int rc = p.vecs == 1 ? (wide ? launch_norm_grad_as<1, true>(h, a, p, st) : launch_norm_grad_as<1, false>(h, a, p, st))
                             : (wide ? launch_norm_grad_as<2, true>(h, a, p, st) : launch_norm_grad_as<2, false>(h, a, p, st));
  if (rc != MG_OK || a.parts == nullptr) return rc;
  norm_grad_sum_kernel<<<static_cast<unsigned>((cols + 31) / 32), 1024, 0, st>>>(a.parts, p.shares, static_cast<int>(cols), gw);
  MG_CUDA(cudaGetLastError());
  return MG_OK;
}

}  // namespace mg
