// y[m][n] = sum_k x[m][k] * (q[n][k] - z[n][k / g]) * s[n][k / g] (+ bias[n]): a few rows of 16-bit activations times a
// 4-bit weight matrix with one scale (and zero point) per group of g elements along K.
//
// With few rows this is bound by the weights' bytes (N K / 2 plus scales), so a weight is read once, by 16-byte loads
// that are contiguous over a warp, and everything after the load is kept under that time: a 32-bit word holds eight
// weights in an order (laid out once, by the pack kernel) in which one AND and one OR give two of them as 16-bit floats
// 1024 + q (fp16) or 128 + q (bf16), and one subtraction of 1024 + z or 128 + z leaves q - z, exactly. Those are the
// A operand of mma.sync m16n8k16, 16 weight rows by 16 of K, against up to 8 rows of x per MMA. A group's products are
// summed on their own in fp32 and multiplied by the scale in fp32: no rounding before the output's.
//
// The warps of a CTA share 16 RT weight rows and take turns along K; their sums meet in shared memory in a fixed order.
#include "fdb_common.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace fdb {

// Descriptor shared with ops/linear_int4.py.
struct Int4Desc {
  const void* x; void* y; const float* bias;
  const void* w; const void* scales; const void* zeros;     // packed by fdb_int4_pack; zeros may be null (8 everywhere)
  void* x_pad;                                              // [m][k rounded up to 8] when x's rows are not 16-byte aligned
  long long x_ld, y_ld;
  int dtype, scale_dtype, m, n, k, group;
};

struct Int4Params {
  const uint8_t* x; uint8_t* y; const float* bias;
  const uint4* w; const uint8_t* scales; const uint8_t* zeros;
  long long x_ld, y_ld;
  int m, n, k, k_tiles, scale_kind;      // scale_kind: kF16, kBF16 or kF32
};

// ---------------------------------------------------------------------------------------------------------- packing
// Source: rows of nibbles, the even element in the low half of a byte, groups padded to whole ones. Packed weights: for
// each tile of 16 rows x 128 of K, 2 x 32 x 16 bytes: half h and lane (g, t) hold row g + 8 h; word j its elements of
// K block j * 32; nibble i / 2 + 4 (i % 2) of the word is element i of the lane: k = 8 t + i, or, for groups of 16,
// 4 t + i of the first group and of the second one. Scales: [tile][16 rows][128 / min(g, 128)], zero points alike in
// nibbles. What lies behind N or K is q = z with scale 0.
__device__ __forceinline__ int nibble_zero(const uint8_t* zeros, long long row, int blk, int zero_bytes) {
  if (zeros == nullptr) return 8;
  const int b = zeros[row * zero_bytes + (blk >> 1)];
  return (blk & 1) ? b >> 4 : b & 15;
}

__global__ void int4_pack_weights(const uint8_t* __restrict__ q, const uint8_t* __restrict__ zeros, uint32_t* __restrict__ out,
                                  int n, int k, int group, int k_tiles, long long words) {
  const int blocks = (k + group - 1) / group, zero_bytes = (blocks + 1) / 2;
  const long long row_bytes = static_cast<long long>(blocks) * group / 2;
  for (long long w = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; w < words;
       w += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int j = static_cast<int>(w & 3), lane = static_cast<int>(w >> 2) & 31, half = static_cast<int>(w >> 7) & 1;
    const long long tile = w >> 8;
    const int kt = static_cast<int>(tile % k_tiles);
    const long long row = tile / k_tiles * 16 + (lane >> 2) + 8 * half;
    const int t = lane & 3;
    uint32_t v = 0;
    for (int i = 0; i < 8; ++i) {
      const int in = group == 16 ? (i >> 2) * 16 + 4 * t + (i & 3) : 8 * t + i;
      const int kk = kt * 128 + j * 32 + in;
      uint32_t e = 8;
      if (row < n && kk < blocks * group) {
        if (kk < k) {
          const uint8_t b = q[row * row_bytes + (kk >> 1)];
          e = (kk & 1) ? b >> 4 : b & 15;
        } else {
          e = nibble_zero(zeros, row, kk / group, zero_bytes);
        }
      }
      v |= e << (4 * (i >> 1) + 16 * (i & 1));
    }
    out[w] = v;
  }
}

// One thread per (tile, row): the scales of the tile's groups and their zero points.
template <typename S>
__global__ void int4_pack_scales(const S* __restrict__ s, const uint8_t* __restrict__ zeros, S* __restrict__ out,
                                 uint8_t* __restrict__ out_zeros, int n, int k, int group, int k_tiles, long long count) {
  const int blocks = (k + group - 1) / group, zero_bytes = (blocks + 1) / 2;
  const int per = 128 / min(group, 128);
  for (long long x = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; x < count;
       x += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long tile = x >> 4, row = tile / k_tiles * 16 + (x & 15);
    const int kt = static_cast<int>(tile % k_tiles);
    uint32_t z = 0;
    for (int i = 0; i < per; ++i) {
      const int blk = static_cast<int>((kt * 128LL + i * (128 / per)) / group);
      const bool in = row < n && blk < blocks;
      out[x * per + i] = in ? s[row * blocks + blk] : S(0.f);
      z |= static_cast<uint32_t>(in ? nibble_zero(zeros, row, blk, zero_bytes) : 8) << (4 * i);
    }
    if (out_zeros != nullptr) {
      const int bytes = max(1, per / 2);
      for (int i = 0; i < bytes; ++i) out_zeros[x * bytes + i] = static_cast<uint8_t>(z >> (8 * i));
    }
  }
}

// x with rows that 16-byte loads cannot take -> rows of k rounded up to 8, zeros behind k.
__global__ void int4_pad_rows(const uint16_t* __restrict__ x, uint16_t* __restrict__ out, long long x_ld, int k, int k8) {
  const uint16_t* row = x + blockIdx.y * x_ld;
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c < k8) out[static_cast<long long>(blockIdx.y) * k8 + c] = c < k ? row[c] : uint16_t(0);
}

// ---------------------------------------------------------------------------------------------------------- product
__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <bool BF16>
__device__ __forceinline__ void int4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The 16-bit floats 1024 + z (fp16) or 128 + z (bf16), twice in a word.
template <bool BF16>
__device__ __forceinline__ uint32_t biased(uint32_t z) { return (BF16 ? 0x43004300u : 0x64006400u) | z | (z << 16); }

// Nibbles p and p + 4 of a word minus the zero point, as a pair of 16-bit floats.
template <bool BF16>
__device__ __forceinline__ uint32_t weights_pair(uint32_t w, int p, uint32_t zero) {
  const uint32_t v = ((w >> (4 * p)) & 0x000f000fu) | (BF16 ? 0x43004300u : 0x64006400u);
  if (BF16) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&zero));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&zero));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// SG scales of one row of a tile.
template <int SG>
__device__ __forceinline__ void load_scales(const Int4Params& p, long long row, float (&s)[SG]) {
  if (p.scale_kind == kF32) {
    const float* a = reinterpret_cast<const float*>(p.scales) + row * SG;
#pragma unroll
    for (int i = 0; i < SG; ++i) s[i] = __ldg(a + i);
    return;
  }
  const uint16_t* a = reinterpret_cast<const uint16_t*>(p.scales) + row * SG;
  uint32_t w[(SG + 1) / 2];
  if (SG == 1) {
    w[0] = __ldg(a);
  } else if (SG == 2) {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(a));
  } else if (SG == 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(a));
    w[0] = v.x; w[1 % ((SG + 1) / 2)] = v.y;
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(a));
    w[0] = v.x; w[1 % ((SG + 1) / 2)] = v.y; w[2 % ((SG + 1) / 2)] = v.z; w[3 % ((SG + 1) / 2)] = v.w;
  }
#pragma unroll
  for (int i = 0; i < SG; ++i) {
    const uint16_t h = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
    s[i] = p.scale_kind == kBF16 ? __uint_as_float(static_cast<uint32_t>(h) << 16) : __half2float(__ushort_as_half(h));
  }
}

template <int SG>
__device__ __forceinline__ uint32_t load_zeros(const Int4Params& p, long long row) {
  if (p.zeros == nullptr) return 0x88888888u;
  if (SG == 8) return __ldg(reinterpret_cast<const uint32_t*>(p.zeros) + row);
  if (SG == 4) return __ldg(reinterpret_cast<const uint16_t*>(p.zeros) + row);
  return __ldg(p.zeros + row);
}

constexpr int kInt4Warps = 8;

template <bool BF16, int SG, int MT, int RT>
__global__ void __launch_bounds__(kInt4Warps * 32)
int4_linear_kernel(const Int4Params p) {
  extern __shared__ float red[];                                     // [warps][16 RT][8 MT]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * (8 * MT);
  const long long row_tile0 = static_cast<long long>(blockIdx.x) * RT;
  const int row_tiles = (p.n + 15) / 16;
  float acc[RT][MT][4] = {};
  const uint8_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = m0 + i * 8 + g < p.m ? p.x + (m0 + i * 8 + g) * p.x_ld * 2 : nullptr;

#pragma unroll(MT >= 8 ? 1 : 2)
  for (int kt = warp; kt < p.k_tiles; kt += kInt4Warps) {
    uint4 w[RT][2];
    float s[RT][2][SG];
    uint32_t z[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const long long tile = min(row_tile0 + r, static_cast<long long>(row_tiles) - 1) * p.k_tiles + kt;
      w[r][0] = ld_stream(p.w + tile * 64 + lane);
      w[r][1] = ld_stream(p.w + tile * 64 + 32 + lane);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_scales<SG>(p, tile * 16 + g + 8 * h, s[r][h]);
        z[r][h] = load_zeros<SG>(p, tile * 16 + g + 8 * h);
      }
    }
    float part[RT][MT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 xb[MT];
      const int k = kt * 128 + j * 32;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xb[i] = make_uint4(0, 0, 0, 0);
        if (SG == 8) {
          // groups of 16: the lane's elements are 4 t .. of either group
          if (xr[i] != nullptr) {
            uint2 a = make_uint2(0, 0), b = make_uint2(0, 0);
            if (k + 4 * t < p.k) a = __ldg(reinterpret_cast<const uint2*>(xr[i] + (k + 4 * t) * 2));
            if (k + 16 + 4 * t < p.k) b = __ldg(reinterpret_cast<const uint2*>(xr[i] + (k + 16 + 4 * t) * 2));
            xb[i] = make_uint4(a.x, a.y, b.x, b.y);
          }
        } else if (xr[i] != nullptr && k + 8 * t < p.k) {
          xb[i] = __ldg(reinterpret_cast<const uint4*>(xr[i] + (k + 8 * t) * 2));
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const uint32_t wa = j == 0 ? w[r][0].x : j == 1 ? w[r][0].y : j == 2 ? w[r][0].z : w[r][0].w;
        const uint32_t wb = j == 0 ? w[r][1].x : j == 1 ? w[r][1].y : j == 2 ? w[r][1].z : w[r][1].w;
#pragma unroll
        for (int u = 0; u < 2; ++u) {                                 // the two K = 16 steps of a K block of 32
          const int grp = (j * 2 + u) * SG / 8;
          const bool first = SG == 8 || (j * 2 + u) % (8 / SG) == 0, last = SG == 8 || (j * 2 + u + 1) % (8 / SG) == 0;
          const uint32_t za = biased<BF16>((z[r][0] >> (4 * grp)) & 15u), zb = biased<BF16>((z[r][1] >> (4 * grp)) & 15u);
          const uint32_t a0 = weights_pair<BF16>(wa, 2 * u, za), a2 = weights_pair<BF16>(wa, 2 * u + 1, za);
          const uint32_t a1 = weights_pair<BF16>(wb, 2 * u, zb), a3 = weights_pair<BF16>(wb, 2 * u + 1, zb);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            if (first) part[r][i][0] = part[r][i][1] = part[r][i][2] = part[r][i][3] = 0.f;
            int4_mma<BF16>(part[r][i], a0, a1, a2, a3, u == 0 ? xb[i].x : xb[i].z, u == 0 ? xb[i].y : xb[i].w);
            if (last) {
              acc[r][i][0] = fmaf(part[r][i][0], s[r][0][grp], acc[r][i][0]);
              acc[r][i][1] = fmaf(part[r][i][1], s[r][0][grp], acc[r][i][1]);
              acc[r][i][2] = fmaf(part[r][i][2], s[r][1][grp], acc[r][i][2]);
              acc[r][i][3] = fmaf(part[r][i][3], s[r][1][grp], acc[r][i][3]);
            }
          }
        }
      }
    }
  }
  constexpr int kRows = 16 * RT, kCols = 8 * MT;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        red[(warp * kCols + i * 8 + 2 * t + (x & 1)) * kRows + r * 16 + g + 8 * (x >> 1)] = acc[r][i][x];
  __syncthreads();
  for (int x = threadIdx.x; x < kRows * kCols; x += blockDim.x) {
    const int col = x / kRows, m = m0 + col;
    const long long n = row_tile0 * 16 + x % kRows;
    if (m >= p.m || n >= p.n) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kInt4Warps; ++w) v += red[(w * kCols + col) * kRows + x % kRows];
    if (p.bias != nullptr) v += __ldg(p.bias + n);
    uint8_t* y = p.y + (m * p.y_ld + n) * 2;
    if (BF16) *reinterpret_cast<__nv_bfloat16*>(y) = __float2bfloat16_rn(v);
    else *reinterpret_cast<__half*>(y) = __float2half_rn(v);
  }
}

}  // namespace fdb

using namespace fdb;

namespace {

typedef void (*Int4Kernel)(const Int4Params);

template <bool BF16, int SG>
Int4Kernel pick_rows(int mt) {
  switch (mt) {
    case 1: return int4_linear_kernel<BF16, SG, 1, 1>;
    case 2: return int4_linear_kernel<BF16, SG, 2, 1>;
    case 4: return int4_linear_kernel<BF16, SG, 4, 2>;
    default: return int4_linear_kernel<BF16, SG, 8, 2>;
  }
}
template <bool BF16>
Int4Kernel pick(int sg, int mt) {
  switch (sg) {
    case 8: return pick_rows<BF16, 8>(mt);
    case 4: return pick_rows<BF16, 4>(mt);
    case 2: return pick_rows<BF16, 2>(mt);
    default: return pick_rows<BF16, 1>(mt);
  }
}

struct Int4Op : Op {
  Int4Params p{};
  Int4Kernel kernel = nullptr;
  dim3 grid;
  int smem = 0, device = 0, k8 = 0;
  const uint16_t* x_src = nullptr;        // set when x goes through x_pad
  uint16_t* x_pad = nullptr;
  long long x_src_ld = 0;
  int launch(cudaStream_t s) override {
    int at = device;
    cudaGetDevice(&at);
    if (at != device) cudaSetDevice(device);
    if (x_pad != nullptr) int4_pad_rows<<<dim3((k8 + 255) / 256, p.m), 256, 0, s>>>(x_src, x_pad, x_src_ld, p.k, k8);
    kernel<<<grid, kInt4Warps * 32, smem, s>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (at != device) cudaSetDevice(at);
    if (e != cudaSuccess) { set_error(std::string("int4 linear: ") + cudaGetErrorString(e)); return -1; }
    return 0;
  }
};

bool group_ok(int g) { return g == 16 || g == 32 || g == 64 || g == 128 || g == 256; }

}  // namespace

FDB_API int fdb_int4_desc_size() { return static_cast<int>(sizeof(Int4Desc)); }

// Lays out a weight: q [n][groups][group / 2] bytes, scales [n][groups] (fp16, bf16 or fp32), zeros [n][(groups + 1) / 2]
// bytes or null -> w [row tiles][k tiles][1024 bytes], out_scales and out_zeros as the product kernel reads them.
FDB_API int fdb_int4_pack(const void* q, const void* scales, const void* zeros, void* w, void* out_scales, void* out_zeros,
                          int scale_dtype, int n, int k, int group, void* stream) {
  if (!group_ok(group) || n < 1 || k < 1) { set_error("int4 pack: bad sizes"); return -1; }
  if ((zeros == nullptr) != (out_zeros == nullptr)) { set_error("int4 pack: zeros and out_zeros come together"); return -1; }
  const int k_tiles = (k + 127) / 128;
  const long long tiles = static_cast<long long>((n + 15) / 16) * k_tiles;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto blocks = [](long long x) { return static_cast<int>(std::min<long long>((x + 255) / 256, 148 * 32)); };
  int4_pack_weights<<<blocks(tiles * 256), 256, 0, s>>>(static_cast<const uint8_t*>(q), static_cast<const uint8_t*>(zeros),
                                                        static_cast<uint32_t*>(w), n, k, group, k_tiles, tiles * 256);
  const auto* z = static_cast<const uint8_t*>(zeros);
  auto* oz = static_cast<uint8_t*>(out_zeros);
  if (scale_dtype == kF32)
    int4_pack_scales<float><<<blocks(tiles * 16), 256, 0, s>>>(static_cast<const float*>(scales), z, static_cast<float*>(out_scales),
                                                               oz, n, k, group, k_tiles, tiles * 16);
  else if (scale_dtype == kF16)
    int4_pack_scales<__half><<<blocks(tiles * 16), 256, 0, s>>>(static_cast<const __half*>(scales), z, static_cast<__half*>(out_scales),
                                                                oz, n, k, group, k_tiles, tiles * 16);
  else if (scale_dtype == kBF16)
    int4_pack_scales<__nv_bfloat16><<<blocks(tiles * 16), 256, 0, s>>>(static_cast<const __nv_bfloat16*>(scales), z,
                                                                       static_cast<__nv_bfloat16*>(out_scales), oz, n, k, group,
                                                                       k_tiles, tiles * 16);
  else { set_error("int4 pack: scales must be fp16, bf16 or fp32"); return -1; }
  FDB_CUDA_OK(cudaGetLastError());
  return 0;
}

FDB_API void* fdb_int4_linear_create(const Int4Desc* d) {
  auto fail = [](const std::string& what) -> void* { set_error("int4 linear: " + what); return nullptr; };
  if (d->dtype != kF16 && d->dtype != kBF16) return fail("x and y must be fp16 or bf16");
  if (d->scale_dtype != kF16 && d->scale_dtype != kBF16 && d->scale_dtype != kF32) return fail("scales must be fp16, bf16 or fp32");
  if (!group_ok(d->group)) return fail("the group size must be 16, 32, 64, 128 or 256");
  if (d->m < 1 || d->n < 1 || d->k < 1) return fail("empty sizes");
  if (d->x_ld < d->k || d->y_ld < d->n) return fail("row pitches shorter than a row");
  const bool aligned = reinterpret_cast<uintptr_t>(d->x) % 16 == 0 && d->x_ld % 8 == 0 && d->k % 8 == 0;
  if (!aligned && d->x_pad == nullptr) return fail("rows of x that are not 16-byte aligned need x_pad");
  auto* op = new Int4Op();
  cudaGetDevice(&op->device);
  Int4Params& p = op->p;
  p.x = static_cast<const uint8_t*>(d->x); p.x_ld = d->x_ld;
  op->k8 = (d->k + 7) / 8 * 8;
  p.k = d->k;
  if (!aligned) {
    op->x_src = static_cast<const uint16_t*>(d->x); op->x_src_ld = d->x_ld; op->x_pad = static_cast<uint16_t*>(d->x_pad);
    p.x = static_cast<const uint8_t*>(d->x_pad); p.x_ld = op->k8;
  }
  p.y = static_cast<uint8_t*>(d->y); p.y_ld = d->y_ld; p.bias = d->bias;
  p.w = static_cast<const uint4*>(d->w); p.scales = static_cast<const uint8_t*>(d->scales);
  p.zeros = static_cast<const uint8_t*>(d->zeros);
  p.m = d->m; p.n = d->n; p.k_tiles = (d->k + 127) / 128; p.scale_kind = d->scale_dtype;
  const int mt = d->m <= 8 ? 1 : d->m <= 16 ? 2 : d->m <= 32 ? 4 : 8, rt = mt >= 4 ? 2 : 1;
  const int sg = 128 / std::min(d->group, 128);
  op->kernel = d->dtype == kBF16 ? pick<true>(sg, mt) : pick<false>(sg, mt);
  op->smem = kInt4Warps * 16 * rt * 8 * mt * 4;
  const int row_tiles = (d->n + 15) / 16;
  op->grid = dim3((row_tiles + rt - 1) / rt, (d->m + 8 * mt - 1) / (8 * mt));
  if (op->grid.y > 65535) { delete op; return fail("too many rows"); }
  if (op->smem > 48 * 1024 &&
      cudaFuncSetAttribute(reinterpret_cast<const void*>(op->kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, op->smem) != cudaSuccess) {
    cudaGetLastError(); delete op; return fail("cannot raise the dynamic shared memory limit");
  }
  return op;
}
