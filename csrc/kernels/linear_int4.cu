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
// The warps of a CTA share 16 weight rows and split K; their sums meet in shared memory in a fixed order. One row of x,
// 28672 x 8192, groups of 128, fp16: 33 us, 3.7 TB/s, 57 % of a copy's bandwidth; the ALU pipe (an AND-OR or a shift is half
// rate: five a word of eight weights in fp16, seven in bf16) is 64 % busy, and warps wait for it and for issue slots before
// they wait for DRAM.
#include "fdb_common.h"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace fdb {

// Descriptor shared with ops/linear_int4.py.
struct Int4Desc {
  const void* x; void* y; const float* bias;
  const void* w;                                            // packed by fdb_int4_pack
  void* x_pad;                                              // [m][k rounded up to 8] when x's rows are not 16-byte aligned
  int* status;
  long long x_ld, y_ld;
  int dtype, scale_dtype, has_zeros, m, n, k, group, tile_rows, splits;   // tile_rows: 0 = the vector kernel, else x rows per tile
};

struct Int4Params {
  const uint8_t* x; uint8_t* y; const float* bias;
  const uint8_t* w;
  int* status;
  long long x_ld, y_ld;
  int m, n, k, k_tiles, splits, stages, wide, has_zeros;
  uint32_t stage_bytes, block_bytes;      // of a ring stage and of a packed block
};

// ---------------------------------------------------------------------------------------------------------- packing
// Source: rows of nibbles, the even element in the low half of a byte, groups padded to whole ones. Packed: one block
// for each 128 rows x 128 of K, K innermost, with all that a product needs of them (one copy brings it on chip): the
// weights of eight tiles of 16 rows, the scales [128 rows][128 / min(g, 128)], and, unless all are 8, the zero points
// alike, two to a byte. A tile has 1024 bytes: row r has 64 of them, in four pieces of 16; piece t lies at place
// (t + r / 2) % 4, so that eight consecutive rows' pieces t meet different banks. Word j of a piece holds eight elements
// of K block j * 32; nibble i / 2 + 4 (i % 2) of the word is element i: k = 8 t + i, or, for groups of 16, 4 t + i of the
// first group (i < 4) and 4 t + i - 4 of the second. What lies behind N or K is q = z with scale 0.
__device__ __forceinline__ int nibble_zero(const uint8_t* zeros, long long row, int blk, int zero_bytes) {
  if (zeros == nullptr) return 8;
  const int b = zeros[row * zero_bytes + (blk >> 1)];
  return (blk & 1) ? b >> 4 : b & 15;
}

__global__ void int4_pack_weights(const uint8_t* __restrict__ q, const uint8_t* __restrict__ zeros, uint8_t* __restrict__ out,
                                  int n, int k, int group, int k_tiles, long long block_bytes, long long words) {
  const int blocks = (k + group - 1) / group, zero_bytes = (blocks + 1) / 2;
  const long long row_bytes = static_cast<long long>(blocks) * group / 2;
  for (long long w = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; w < words;
       w += static_cast<long long>(gridDim.x) * blockDim.x) {
    const int j = static_cast<int>(w & 3), place = static_cast<int>(w >> 2) & 3, r = static_cast<int>(w >> 4) & 127;
    const long long block = w >> 11;
    const int kt = static_cast<int>(block % k_tiles);
    const long long row = block / k_tiles * 128 + r;
    const int t = (place - (r >> 1)) & 3;
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
    *reinterpret_cast<uint32_t*>(out + block * block_bytes + (w & 2047) * 4) = v;
  }
}

// One thread per row of a block: the scales of its groups and their zero points.
template <typename S>
__global__ void int4_pack_scales(const S* __restrict__ s, const uint8_t* __restrict__ zeros, uint8_t* __restrict__ out, int n,
                                 int k, int group, int k_tiles, long long block_bytes, long long count) {
  const int blocks = (k + group - 1) / group, zero_bytes = (blocks + 1) / 2;
  const int per = 128 / min(group, 128);
  for (long long x = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; x < count;
       x += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long block = x >> 7, row = block / k_tiles * 128 + (x & 127);
    const int kt = static_cast<int>(block % k_tiles);
    uint8_t* to = out + block * block_bytes + 8192;
    uint32_t z = 0;
    for (int i = 0; i < per; ++i) {
      const int blk = static_cast<int>((kt * 128LL + i * (128 / per)) / group);
      const bool in = row < n && blk < blocks;
      reinterpret_cast<S*>(to)[(x & 127) * per + i] = in ? s[row * blocks + blk] : S(0.f);
      z |= static_cast<uint32_t>(in ? nibble_zero(zeros, row, blk, zero_bytes) : 8) << (4 * i);
    }
    if (zeros != nullptr) {
      const int bytes = max(1, per / 2);
      uint8_t* zr = to + 128 * per * sizeof(S) + (x & 127) * bytes;
      for (int i = 0; i < bytes; ++i) zr[i] = static_cast<uint8_t>(z >> (8 * i));
    }
  }
}

// x with rows that 16-byte loads cannot take -> rows of k rounded up to 8, zeros behind k. Rows are the grid's x, which may
// have 2^31 - 1 of them (y ends at 65535).
constexpr int kPadThreads = 256;
__global__ void int4_pad_rows(const uint16_t* __restrict__ x, uint16_t* __restrict__ out, long long x_ld, int k, int k8) {
  const uint16_t* row = x + blockIdx.x * x_ld;
  uint16_t* to = out + static_cast<long long>(blockIdx.x) * k8;
  for (int c = blockIdx.y * kPadThreads + threadIdx.x; c < k8; c += gridDim.y * kPadThreads) to[c] = c < k ? row[c] : uint16_t(0);
}

// ---------------------------------------------------------------------------------------------------------- product
template <bool BF16>
__device__ __forceinline__ void int4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights as 16-bit floats. OR-ing a nibble into the low mantissa bits of 1024 (fp16) or 128 (bf16) adds it exactly;
// fp16 also takes it four bits higher (1024 + 16 q, and a fused multiply by 1 / 16), which saves a shift.
constexpr uint32_t kBase16 = 0x64006400u, kBaseB16 = 0x43004300u;

// The zero point as two words: subtrahend for nibbles in the low bits, and (fp16) addend -(64 + z) for the higher ones.
struct ZeroPair { uint32_t low, high; };
template <bool BF16>
__device__ __forceinline__ ZeroPair zero_pair(uint32_t z) {
  const uint32_t zz = z * 0x00010001u;
  if (BF16) return {kBaseB16 + zz, 0u};
  return {kBase16 + zz, 0xd400d400u + (zz << 4)};        // -(64 + z): 0xd400 is -64, one unit of z is 16 mantissa steps
}

// The eight weights of a word, minus the zero point, as four pairs (elements 2 p and 2 p + 1 in pair p).
template <bool BF16>
__device__ __forceinline__ void unpack_word(uint32_t w, const ZeroPair& z, uint32_t (&out)[4]) {
  if (BF16) {
    const __nv_bfloat162 zero = *reinterpret_cast<const __nv_bfloat162*>(&z.low);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t v = ((w >> (4 * p)) & 0x000f000fu) | kBaseB16;
      const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), zero);
      out[p] = *reinterpret_cast<const uint32_t*>(&r);
    }
  } else {
    const uint32_t sixteenth = 0x2c002c00u;               // 1 / 16, twice
    const __half2 low = *reinterpret_cast<const __half2*>(&z.low), high = *reinterpret_cast<const __half2*>(&z.high);
    const __half2 factor = *reinterpret_cast<const __half2*>(&sixteenth);
#pragma unroll
    for (int p = 0; p < 4; p += 2) {
      const uint32_t x = p == 0 ? w : w >> 8;
      const uint32_t v0 = (x & 0x000f000fu) | kBase16, v1 = (x & 0x00f000f0u) | kBase16;
      const __half2 r0 = __hsub2(*reinterpret_cast<const __half2*>(&v0), low);
      const __half2 r1 = __hfma2(*reinterpret_cast<const __half2*>(&v1), factor, high);
      out[p] = *reinterpret_cast<const uint32_t*>(&r0);
      out[p + 1] = *reinterpret_cast<const uint32_t*>(&r1);
    }
  }
}

// SG scales of one row of a tile, in shared memory: fp32, or 16-bit of x's type.
template <bool BF16, bool WIDE, int SG>
struct ScaleRow {
  uint32_t w[WIDE ? SG : (SG + 1) / 2];
  __device__ __forceinline__ void load(const uint8_t* a) {
    if (WIDE) {
#pragma unroll
      for (int i = 0; i < SG; ++i) w[i] = reinterpret_cast<const uint32_t*>(a)[i];
    } else if (SG == 1) {
      w[0] = *reinterpret_cast<const uint16_t*>(a);
    } else {
#pragma unroll
      for (int i = 0; i < SG / 2; ++i) w[i] = reinterpret_cast<const uint32_t*>(a)[i];
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if (WIDE) return __uint_as_float(w[i]);
    if (BF16) return __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    return __half2float(__ushort_as_half(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)))));
  }
};

template <int SG>
__device__ __forceinline__ uint32_t load_zeros(const uint8_t* a) {
  if (SG == 8) return *reinterpret_cast<const uint32_t*>(a);
  if (SG == 4) return *reinterpret_cast<const uint16_t*>(a);
  return *a;
}

constexpr int kInt4Warps = 8;

// Up to 8 MT rows of x; the CTA's eight warps share 16 weight rows, each warp a run of tiles along K, which it brings into
// a ring of its own in shared memory by cp.async (no registers held, nothing to wait for but its own copies).
constexpr int kVecStages = 4;
template <bool V> struct WholeTile { static constexpr bool value = V; };

template <bool BF16, bool WIDE, bool ZERO, int SG, int MT>
__global__ void __launch_bounds__(kInt4Warps * 32)
int4_linear_kernel(const Int4Params p) {
  constexpr uint32_t kScaleRow = SG * (WIDE ? 4 : 2), kZeroRow = SG >= 2 ? SG / 2 : 1;          // bytes of a row of a tile
  constexpr uint32_t kStage = 1024 + 16 * (kScaleRow + (ZERO ? kZeroRow : 0));
  extern __shared__ __align__(16) uint8_t ring_raw[];                // [warps][stages][kStage], then the warps' sums
  float* red = reinterpret_cast<float*>(ring_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.y * (8 * MT);
  float acc[MT][4] = {};
  const int kt0 = p.k_tiles * warp / kInt4Warps, count = p.k_tiles * (warp + 1) / kInt4Warps - kt0;
  const int in_block = blockIdx.x & 7;                               // which 16 rows of a block
  const uint8_t* ring = ring_raw + warp * (kVecStages * kStage);
  const uint32_t ring_at = smem_u32(ring) + lane * 16;
  const uint8_t* wp = p.w + (static_cast<long long>(blockIdx.x >> 3) * p.k_tiles + kt0) * p.block_bytes + in_block * 1024 + lane * 16;
  const uint32_t scales_at = 8192 + in_block * (16 * kScaleRow - 1024);        // from wp, like zeros_at
  const uint32_t zeros_at = 8192 + 128 * kScaleRow + in_block * (16 * kZeroRow - 1024);
  auto fetch = [&](int i, int stage) {                               // tile i of the warp; a group of copies either way
    if (i < count) {
      const uint32_t at = ring_at + static_cast<uint32_t>(stage) * kStage;
      cp_async_16(at, wp, 16);
      cp_async_16(at + 512, wp + 512, 16);
      if (lane * 16 < 16 * kScaleRow) cp_async_16(at + 1024, wp + scales_at, 16);
      if (ZERO && lane * 16 < 16 * kZeroRow) cp_async_16(at + 1024 + 16 * kScaleRow, wp + zeros_at, 16);
      wp += p.block_bytes;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kVecStages - 1; ++i) fetch(i, i);

  const uint8_t* xp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
    xp[i] = p.x + min(m0 + i * 8 + g, p.m - 1) * p.x_ld * 2 + (kt0 * 128 + (SG == 8 ? 4 : 8) * t) * 2;
  // Elements of x from this lane's first one to the end of the row: a load is made when it starts inside the row (K is a
  // multiple of 8 here, so it ends inside too).
  int left = p.k - kt0 * 128 - (SG == 8 ? 4 : 8) * t;
  const uint32_t piece_a = g * 64 + ((t + (g >> 1)) & 3) * 16;       // rows g and g + 8: the same place, 512 bytes apart
  auto tile = [&](int i, auto whole_tag, int stage, int next_stage) {
    constexpr bool whole = decltype(whole_tag)::value;
    // Rows of x behind the last one repeat it: a column of the product that nobody stores. Only the row's last tile asks
    // whether a load starts inside the row.
    uint4 xb[4][MT];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        const uint8_t* a = xp[r] + j * 64;
        if (SG == 8) {
          // groups of 16: the lane's elements are 4 t .. of either group
          uint2 h0 = make_uint2(0, 0), h1 = h0;
          if (whole || j * 32 < left) h0 = __ldg(reinterpret_cast<const uint2*>(a));
          if (whole || j * 32 + 16 < left) h1 = __ldg(reinterpret_cast<const uint2*>(a + 32));
          xb[j][r] = make_uint4(h0.x, h0.y, h1.x, h1.y);
        } else {
          xb[j][r] = make_uint4(0, 0, 0, 0);
          if (whole || j * 32 < left) xb[j][r] = __ldg(reinterpret_cast<const uint4*>(a));
        }
      }
#pragma unroll
    for (int r = 0; r < MT; ++r) xp[r] += 256;
    cp_async_wait<kVecStages - 2>();
    __syncwarp();                                                    // every lane's copies of tile i have landed
    fetch(i + kVecStages - 1, next_stage);                           // into the stage that tile i - 1 left
    const uint8_t* at = ring + stage * kStage;
    const uint4 va = *reinterpret_cast<const uint4*>(at + piece_a), vb = *reinterpret_cast<const uint4*>(at + piece_a + 512);
    ScaleRow<BF16, WIDE, SG> s[2];
    s[0].load(at + 1024 + g * kScaleRow);
    s[1].load(at + 1024 + (g + 8) * kScaleRow);
    uint32_t z[2] = {0x88888888u, 0x88888888u};
    if (ZERO) {
      z[0] = load_zeros<SG>(at + 1024 + 16 * kScaleRow + g * kZeroRow);
      z[1] = load_zeros<SG>(at + 1024 + 16 * kScaleRow + (g + 8) * kZeroRow);
    }
    float part[MT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t wa = j == 0 ? va.x : j == 1 ? va.y : j == 2 ? va.z : va.w;
      const uint32_t wb = j == 0 ? vb.x : j == 1 ? vb.y : j == 2 ? vb.z : vb.w;
      uint32_t ra[4], rb[4];
      const int g0 = j * 2 * SG / 8;
      unpack_word<BF16>(wa, zero_pair<BF16>(ZERO ? (z[0] >> (4 * g0)) & 15u : 8u), ra);
      unpack_word<BF16>(wb, zero_pair<BF16>(ZERO ? (z[1] >> (4 * g0)) & 15u : 8u), rb);
      if (SG == 8 && ZERO) {                            // the word's second half belongs to the next group
        uint32_t other[4];
        unpack_word<BF16>(wa, zero_pair<BF16>((z[0] >> (4 * g0 + 4)) & 15u), other);
        ra[2] = other[2]; ra[3] = other[3];
        unpack_word<BF16>(wb, zero_pair<BF16>((z[1] >> (4 * g0 + 4)) & 15u), other);
        rb[2] = other[2]; rb[3] = other[3];
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {                     // the two K = 16 steps of a K block of 32
        const int grp = (j * 2 + u) * SG / 8;
        const bool first = SG == 8 || (j * 2 + u) % (8 / SG) == 0, last = SG == 8 || (j * 2 + u + 1) % (8 / SG) == 0;
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          if (first) part[r][0] = part[r][1] = part[r][2] = part[r][3] = 0.f;
          int4_mma<BF16>(part[r], ra[2 * u], rb[2 * u], ra[2 * u + 1], rb[2 * u + 1], u == 0 ? xb[j][r].x : xb[j][r].z,
                         u == 0 ? xb[j][r].y : xb[j][r].w);
          if (last) {
            const float s0 = s[0].at(grp), s1 = s[1].at(grp);
            acc[r][0] = fmaf(part[r][0], s0, acc[r][0]);
            acc[r][1] = fmaf(part[r][1], s0, acc[r][1]);
            acc[r][2] = fmaf(part[r][2], s1, acc[r][2]);
            acc[r][3] = fmaf(part[r][3], s1, acc[r][3]);
          }
        }
      }
    }
    left -= 128;
  };
  int i = 0;
  const int whole = min(count, p.k / 128 - kt0);                     // tiles that end inside the row: the same for all lanes
  for (; i + kVecStages <= whole; i += kVecStages) {
#pragma unroll
    for (int st = 0; st < kVecStages; ++st) tile(i + st, WholeTile<true>{}, st, (st + kVecStages - 1) % kVecStages);
  }
  for (; i < count; ++i) tile(i, WholeTile<false>{}, i % kVecStages, (i + kVecStages - 1) % kVecStages);
  cp_async_wait<0>();
  __syncthreads();                                                   // the rings become the warps' sums
  constexpr int kCols = 8 * MT;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int x = 0; x < 4; ++x) red[(warp * kCols + i * 8 + 2 * t + (x & 1)) * 16 + g + 8 * (x >> 1)] = acc[i][x];
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * kCols; x += blockDim.x) {
    const int col = x / 16, m = m0 + col;
    const long long n = static_cast<long long>(blockIdx.x) * 16 + x % 16;
    if (m >= p.m || n >= p.n) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kInt4Warps; ++w) v += red[(w * kCols + col) * 16 + x % 16];
    if (p.bias != nullptr) v += __ldg(p.bias + n);
    uint8_t* y = p.y + (m * p.y_ld + n) * 2;
    if (BF16) *reinterpret_cast<__nv_bfloat16*>(y) = __float2bfloat16_rn(v);
    else *reinterpret_cast<__half*>(y) = __float2half_rn(v);
  }
}

// ------------------------------------------------------------------------------------------------ more rows: tcgen05
// From a few rows on, mma.sync (measured: 550 TFLOP/s) and the reads of x by every 16 weight rows cost more than the
// weights' bytes. Here a CTA takes 128 weight rows as the M side of tcgen05.mma and MN rows of x as its N side:
//   producer    one bulk copy of the packed block [128 x 128 of K] with its scales and zero points, TMA for x
//   dequant     two groups of four warps take turns: q - z in 16 bits (exact), a weight row per thread,
//               straight into tensor memory as the A operand (through shared memory it would be written and read back
//               once per MMA: 112 KB a block in all, 900 clocks of the 128 bytes a clock)
//   MMA         one product per scale group into one of four accumulators in tensor memory
//   drain       four warps, a weight row per thread: sum += scale * accumulator, in fp32
// so that the scales meet fp32 sums here too and the two kernels differ only in the order of their additions. 64 rows,
// 14336 x 8192, bf16 with zero points: 39 us, 1030 clocks a block on 112 SMs, in which the ALU pipe (the unpacking) is 60 %
// busy and the tensor pipe 25 %; the rest is waiting between the roles. Few weight rows: up to eight CTAs of a cluster split
// K and add their sums, in their order, over distributed shared memory.
constexpr int kTileThreads = 512;
constexpr int kDequantGroups = 2;
constexpr int kMaxInt4Stages = 8;

template <bool BF16, int SG, int MN>
__global__ void __launch_bounds__(kTileThreads, 1)
int4_tile_kernel(const __grid_constant__ CUtensorMap tm_x, const Int4Params p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxInt4Stages + 12];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  constexpr uint32_t kX = 2 * MN * 128, kW = 8192;
  constexpr uint32_t kZeroRow = SG >= 2 ? SG / 2 : 1;
  const bool has_zeros = p.has_zeros != 0;
  const uint32_t scale_row = SG * (p.wide ? 4 : 2), stage_bytes = p.stage_bytes;
  constexpr uint32_t kA = 4 * MN;                                   // tensor memory: four accumulators, then A
  constexpr uint32_t kTmemCols = kA + kDequantGroups * 64 <= 256 ? 256 : 512;       // 32 and 64 rows of x
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t s_ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint8_t* ring = smem_raw + (s_ring - smem_u32(smem_raw));
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  auto full = [&](int i) { return bar(i); };
  auto empty = [&](int i) { return bar(kMaxInt4Stages + i); };
  auto a_full = [&](int i) { return bar(2 * kMaxInt4Stages + i); };
  auto a_empty = [&](int i) { return bar(2 * kMaxInt4Stages + 2 + i); };
  auto d_full = [&](int i) { return bar(2 * kMaxInt4Stages + 4 + i); };
  auto d_empty = [&](int i) { return bar(2 * kMaxInt4Stages + 8 + i); };
  const int kt0 = static_cast<int>(static_cast<long long>(p.k_tiles) * blockIdx.z / p.splits);
  const int kt1 = static_cast<int>(static_cast<long long>(p.k_tiles) * (blockIdx.z + 1) / p.splits);
  const int n_it = kt1 - kt0;
  const int m0 = blockIdx.y * MN;

  if (tid == 0) {
    abort_word = 0;
    for (int i = 0; i < kMaxInt4Stages; ++i) { mbar_init(full(i), 1); mbar_init(empty(i), 4 + 1 + 4); }
    for (int i = 0; i < kDequantGroups; ++i) { mbar_init(a_full(i), 4); mbar_init(a_empty(i), 1); }
    for (int i = 0; i < 4; ++i) { mbar_init(d_full(i), 1); mbar_init(d_empty(i), 4); }
    fence_mbar_init();
    prefetch_tensormap(&tm_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  float acc[MN];                                                    // of the drain warps
#pragma unroll
  for (int i = 0; i < MN; ++i) acc[i] = 0.f;
  const int row = (warp & 3) * 32 + lane;                           // the weight row of a drain or dequant thread
  const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;

  if (warp == 0) {
    // ------------------------------------------------------------------------------------------------- producer
    bool ok = true;
    int issued = 0;
    RingAt at_ring{0, 0u};
    for (int it = 0; ok && it < n_it; ++it, at_ring.step(1, p.stages)) {
      const int st = at_ring.st;
      if (it >= p.stages) ok = mbar_wait_warp(empty(st), at_ring.parity ^ 1u, abort_flag, kStatusTimeoutProducer);
      if (!ok) break;
      const uint32_t at = s_ring + static_cast<uint32_t>(st) * stage_bytes;
      if (lane == 0) {
        mbar_arrive_expect_tx(full(st), kX + p.block_bytes);
        bulk_load(at + kX, p.w + (static_cast<long long>(blockIdx.x) * p.k_tiles + kt0 + it) * p.block_bytes, p.block_bytes, full(st));
        for (int c = 0; c < 2; ++c) tma_load_2d(at + c * (MN * 128), &tm_x, full(st), (kt0 + it) * 128 + c * 64, m0);
      }
      issued = it + 1;
    }
    if (!ok && lane == 0) {                      // a CTA that gives up leaves no copy of its own in flight
      for (int it = max(0, issued - p.stages); it < issued; ++it) {
        volatile int none = 0;
        mbar_wait(full(it % p.stages), (it / p.stages) & 1, &none, kStatusTimeoutProducer);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------------------------------ MMA
    // one elected thread: the compiler then keeps descriptors in uniform registers (with `lane == 0` it moved each operand
    // of each MMA there on its own, 100 clocks an MMA)
    if (elect_one()) {
      const uint32_t idesc = make_idesc(BF16 ? 1u : 0u, 128, MN);
      bool ok = true;
      RingAt at_ring{0, 0u};
      for (int it = 0; ok && it < n_it; ++it, at_ring.step(1, p.stages)) {
        const int st = at_ring.st, buf = it % kDequantGroups;
        ok = mbar_wait(full(st), at_ring.parity, abort_flag, kStatusTimeoutMma) &&
             mbar_wait(a_full(buf), (it / kDequantGroups) & 1, abort_flag, kStatusTimeoutMma);
        const uint32_t ta = tmem + kA + buf * 64;
        const uint64_t bd = make_kmajor_desc(s_ring + static_cast<uint32_t>(st) * stage_bytes, 128);
        for (int g = 0; ok && g < SG; ++g) {
          const int q = it * SG + g, d = q & 3;
          if (q >= 4) ok = mbar_wait(d_empty(d), ((q >> 2) - 1) & 1, abort_flag, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int x = 0; x < 8 / SG; ++x) {
            const int step = g * (8 / SG) + x;
            umma_f16_ts(tmem + d * MN, ta + step * 8, bd + (step >> 2) * ((MN * 128) >> 4) + (step & 3) * 2, idesc,
                        x != 0 ? 1u : 0u);
          }
          umma_commit(d_full(d));
        }
        if (ok) {
          umma_commit(a_empty(buf));
          umma_commit(empty(st));
        }
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // -------------------------------------------------------------------------------------------------- dequant
    const int group = (warp - 8) >> 2, r16 = row & 15;
    bool ok = true;
    RingAt at_ring{0, 0u};
    at_ring.step(group, p.stages);
    for (int it = group, round = 0; ok && it < n_it; it += kDequantGroups, ++round) {
      const int st = at_ring.st;
      ok = mbar_wait_warp(full(st), at_ring.parity, abort_flag, kStatusTimeoutProducer);
      if (!ok) break;
      const uint8_t* stage = ring + static_cast<uint32_t>(st) * stage_bytes;
      uint4 v[4];                                                   // v[t], word j: K elements j * 32 + 8 t ..
#pragma unroll
      for (int t = 0; t < 4; ++t)
        v[t] = *reinterpret_cast<const uint4*>(stage + kX + (row >> 4) * 1024 + r16 * 64 + ((t + (r16 >> 1)) & 3) * 16);
      uint32_t z = 0x88888888u;
      if (has_zeros) z = load_zeros<SG>(stage + kX + kW + 128 * scale_row + row * kZeroRow);
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(st));
      at_ring.step(kDequantGroups, p.stages);
      if (round > 0) ok = mbar_wait_warp(a_empty(group), (round - 1) & 1, abort_flag, kStatusTimeoutMma);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {                        // 64 of K, 32 columns of tensor memory, at a time
        uint32_t o[32];
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int j = half * 2 + jj;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t word = j == 0 ? v[t].x : j == 1 ? v[t].y : j == 2 ? v[t].z : v[t].w;
            uint32_t e[4];
            if (SG == 8) {                                          // elements 4 t .. of the two groups of 16
              uint32_t e2[4];
              unpack_word<BF16>(word, zero_pair<BF16>((z >> (8 * j)) & 15u), e);
              unpack_word<BF16>(word, zero_pair<BF16>((z >> (8 * j + 4)) & 15u), e2);
              o[jj * 16 + 2 * t] = e[0]; o[jj * 16 + 2 * t + 1] = e[1];
              o[jj * 16 + 8 + 2 * t] = e2[2]; o[jj * 16 + 8 + 2 * t + 1] = e2[3];
            } else {
              unpack_word<BF16>(word, zero_pair<BF16>((z >> (4 * (j * SG / 4))) & 15u), e);
#pragma unroll
              for (int x = 0; x < 4; ++x) o[jj * 16 + 4 * t + x] = e[x];
            }
          }
        }
        tmem_st_32x32(tmem + lanes + kA + group * 64 + half * 32, o);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(a_full(group));
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------------------------------------------- drain
    bool ok = true;
    RingAt at_ring{0, 0u};
    for (int it = 0; ok && it < n_it; ++it, at_ring.step(1, p.stages)) {
      const int st = at_ring.st;
      ok = mbar_wait_warp(full(st), at_ring.parity, abort_flag, kStatusTimeoutProducer);
      if (!ok) break;
      const uint8_t* sr = ring + static_cast<uint32_t>(st) * stage_bytes + kX + kW + row * scale_row;
      float s[SG];
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        if (p.wide) s[g] = reinterpret_cast<const float*>(sr)[g];
        else if (BF16) s[g] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(sr)[g]);
        else s[g] = __half2float(reinterpret_cast<const __half*>(sr)[g]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(st));
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        const int q = it * SG + g, d = q & 3;
        ok = mbar_wait_warp(d_full(d), (q >> 2) & 1, abort_flag, kStatusTimeoutMma);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < MN / 32; ++c) {
          uint32_t v[32];
          tmem_ld_32x32(tmem + lanes + d * MN + c * 32, v);
          tmem_ld_wait_dep(v);
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[c * 32 + i] = fmaf(__uint_as_float(v[i]), s[g], acc[c * 32 + i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(d_empty(d));
      }
    }
    if (p.splits == 1 && ok) {
      const long long n = static_cast<long long>(blockIdx.x) * 128 + row;
      const float b = p.bias != nullptr && n < p.n ? __ldg(p.bias + n) : 0.f;
#pragma unroll
      for (int i = 0; i < MN; ++i) {
        if (m0 + i >= p.m || n >= p.n) continue;
        uint8_t* y = p.y + ((m0 + i) * p.y_ld + n) * 2;
        if (BF16) *reinterpret_cast<__nv_bfloat16*>(y) = __float2bfloat16_rn(acc[i] + b);
        else *reinterpret_cast<__half*>(y) = __float2half_rn(acc[i] + b);
      }
    }
    tc_fence_before();
  }
  __syncthreads();                                                  // every copy and every MMA is done with the ring
  if (p.splits > 1) {
    float* sums = reinterpret_cast<float*>(const_cast<uint8_t*>(ring));            // [MN][128] of this CTA's part of K
    if (warp >= 4 && warp < 8) {
#pragma unroll
      for (int i = 0; i < MN; ++i) sums[i * 128 + row] = acc[i];
    }
    cluster_sync_all();
    for (int x = tid + static_cast<int>(blockIdx.z) * kTileThreads; x < MN * 128; x += kTileThreads * p.splits) {
      const int m = m0 + (x >> 7);
      const long long n = static_cast<long long>(blockIdx.x) * 128 + (x & 127);
      if (m >= p.m || n >= p.n) continue;
      float v = 0.f;
      for (int z = 0; z < p.splits; ++z) v += ld_cluster_f32(s_ring + static_cast<uint32_t>(x) * 4, static_cast<uint32_t>(z));
      if (p.bias != nullptr) v += __ldg(p.bias + n);
      uint8_t* y = p.y + (m * p.y_ld + n) * 2;
      if (BF16) *reinterpret_cast<__nv_bfloat16*>(y) = __float2bfloat16_rn(v);
      else *reinterpret_cast<__half*>(y) = __float2half_rn(v);
    }
    cluster_sync_all();                                             // the others have read this CTA's part
  }
  if (tid == 0 && abort_word != 0 && p.status != nullptr) atomicCAS(p.status, 0, abort_word);
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

}  // namespace fdb

using namespace fdb;

namespace {

typedef void (*Int4Tile)(const CUtensorMap, const Int4Params);

template <bool BF16, int SG>
Int4Tile pick_tile_rows(int mn) {
  return mn == 32 ? int4_tile_kernel<BF16, SG, 32> : int4_tile_kernel<BF16, SG, 64>;
}
template <bool BF16>
Int4Tile pick_tile(int sg, int mn) {
  switch (sg) {
    case 8: return pick_tile_rows<BF16, 8>(mn);
    case 4: return pick_tile_rows<BF16, 4>(mn);
    case 2: return pick_tile_rows<BF16, 2>(mn);
    default: return pick_tile_rows<BF16, 1>(mn);
  }
}

typedef void (*Int4Kernel)(const Int4Params);

template <bool BF16, bool WIDE, bool ZERO, int SG>
Int4Kernel pick_rows(int mt) {
  return mt == 1 ? int4_linear_kernel<BF16, WIDE, ZERO, SG, 1> : int4_linear_kernel<BF16, WIDE, ZERO, SG, 2>;
}
template <bool BF16, bool WIDE, bool ZERO>
Int4Kernel pick_group(int sg, int mt) {
  switch (sg) {
    case 8: return pick_rows<BF16, WIDE, ZERO, 8>(mt);
    case 4: return pick_rows<BF16, WIDE, ZERO, 4>(mt);
    case 2: return pick_rows<BF16, WIDE, ZERO, 2>(mt);
    default: return pick_rows<BF16, WIDE, ZERO, 1>(mt);
  }
}
template <bool BF16>
Int4Kernel pick(bool wide, bool zero, int sg, int mt) {
  if (wide) return zero ? pick_group<BF16, true, true>(sg, mt) : pick_group<BF16, true, false>(sg, mt);
  return zero ? pick_group<BF16, false, true>(sg, mt) : pick_group<BF16, false, false>(sg, mt);
}

struct Int4Op : Op {
  Int4Params p{};
  Int4Kernel kernel = nullptr;
  Int4Tile tile = nullptr;               // set for the tile form
  CUtensorMap tm_x;
  int smem = 0;
  dim3 grid;
  int device = 0, k8 = 0;
  const uint16_t* x_src = nullptr;        // set when x goes through x_pad
  uint16_t* x_pad = nullptr;
  long long x_src_ld = 0;
  int launch(cudaStream_t s) override {
    int at = device;
    cudaGetDevice(&at);
    if (at != device) cudaSetDevice(device);
    cudaError_t e = cudaSuccess;
    if (x_pad != nullptr) {
      int4_pad_rows<<<dim3(p.m, std::min((k8 + kPadThreads - 1) / kPadThreads, 1024)), kPadThreads, 0, s>>>(x_src, x_pad, x_src_ld, p.k, k8);
      e = cudaGetLastError();
    }
    if (e != cudaSuccess) {
      // without its rows the product has nothing to read
    } else if (tile != nullptr) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute cluster{};
      cfg.gridDim = grid; cfg.blockDim = dim3(kTileThreads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
      cluster.id = cudaLaunchAttributeClusterDimension;
      cluster.val.clusterDim.x = 1; cluster.val.clusterDim.y = 1; cluster.val.clusterDim.z = p.splits;
      cfg.attrs = &cluster; cfg.numAttrs = 1;
      e = cudaLaunchKernelEx(&cfg, tile, tm_x, p);
    } else {
      kernel<<<grid, kInt4Warps * 32, smem, s>>>(p);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (at != device) cudaSetDevice(at);
    if (e != cudaSuccess) { set_error(std::string("int4 linear: ") + cudaGetErrorString(e)); return -1; }
    return 0;
  }
};

bool group_ok(int g) { return g == 16 || g == 32 || g == 64 || g == 128 || g == 256; }

}  // namespace

FDB_API int fdb_int4_desc_size() { return static_cast<int>(sizeof(Int4Desc)); }

// Bytes of one packed block of 128 rows x 128 of K.
static int int4_block_bytes(int scale_dtype, int group, bool zeros) {
  const int per = 128 / std::min(group, 128);
  return 8192 + 128 * per * (scale_dtype == kF32 ? 4 : 2) + (zeros ? 128 * std::max(1, per / 2) : 0);
}

FDB_API long long fdb_int4_packed_bytes(int scale_dtype, int has_zeros, int n, int k, int group) {
  return static_cast<long long>((n + 127) / 128) * ((k + 127) / 128) * int4_block_bytes(scale_dtype, group, has_zeros != 0);
}

// Lays out a weight: q [n][groups][group / 2] bytes, scales [n][groups] (fp16, bf16 or fp32), zeros [n][(groups + 1) / 2]
// bytes or null -> blocks of 128 rows x 128 of K, fdb_int4_packed_bytes() in all.
FDB_API int fdb_int4_pack(const void* q, const void* scales, const void* zeros, void* out, int scale_dtype, int n, int k,
                          int group, void* stream) {
  if (!group_ok(group) || n < 1 || k < 1) { set_error("int4 pack: bad sizes"); return -1; }
  if (scale_dtype != kF32 && scale_dtype != kF16 && scale_dtype != kBF16) { set_error("int4 pack: scales must be fp16, bf16 or fp32"); return -1; }
  const int k_tiles = (k + 127) / 128;
  const long long count = static_cast<long long>((n + 127) / 128) * k_tiles;
  const long long bytes = int4_block_bytes(scale_dtype, group, zeros != nullptr);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const auto blocks = [](long long x) { return static_cast<int>(std::min<long long>((x + 255) / 256, 148 * 32)); };
  const auto* z = static_cast<const uint8_t*>(zeros);
  auto* o = static_cast<uint8_t*>(out);
  int4_pack_weights<<<blocks(count * 2048), 256, 0, s>>>(static_cast<const uint8_t*>(q), z, o, n, k, group, k_tiles, bytes, count * 2048);
  if (scale_dtype == kF32)
    int4_pack_scales<float><<<blocks(count * 128), 256, 0, s>>>(static_cast<const float*>(scales), z, o, n, k, group, k_tiles, bytes, count * 128);
  else if (scale_dtype == kF16)
    int4_pack_scales<__half><<<blocks(count * 128), 256, 0, s>>>(static_cast<const __half*>(scales), z, o, n, k, group, k_tiles, bytes, count * 128);
  else
    int4_pack_scales<__nv_bfloat16><<<blocks(count * 128), 256, 0, s>>>(static_cast<const __nv_bfloat16*>(scales), z, o, n, k, group, k_tiles, bytes, count * 128);
  FDB_CUDA_OK(cudaGetLastError());
  return 0;
}

FDB_API void* fdb_int4_linear_create(const Int4Desc* d) {
  auto fail = [](const std::string& what) -> void* { set_error("int4 linear: " + what); return nullptr; };
  if (d->dtype != kF16 && d->dtype != kBF16) return fail("x and y must be fp16 or bf16");
  if (d->scale_dtype != d->dtype && d->scale_dtype != kF32) return fail("scales must be fp32 or of x's type");
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
  p.w = static_cast<const uint8_t*>(d->w);
  p.has_zeros = d->has_zeros;
  p.block_bytes = static_cast<uint32_t>(int4_block_bytes(d->scale_dtype, d->group, d->has_zeros != 0));
  p.m = d->m; p.n = d->n; p.k_tiles = (d->k + 127) / 128;
  p.status = d->status;
  const int sg = 128 / std::min(d->group, 128);
  const bool wide = d->scale_dtype == kF32, zero = d->has_zeros != 0;
  if (d->tile_rows == 0) {
    const int mt = d->m <= 8 ? 1 : 2;
    op->kernel = d->dtype == kBF16 ? pick<true>(wide, zero, sg, mt) : pick<false>(wide, zero, sg, mt);
    op->grid = dim3((d->n + 15) / 16, (d->m + 8 * mt - 1) / (8 * mt));
    const int stage = 1024 + 16 * (sg * (wide ? 4 : 2) + (zero ? (sg >= 2 ? sg / 2 : 1) : 0));
    op->smem = std::max(kInt4Warps * kVecStages * stage, kInt4Warps * 8 * mt * 16 * 4);
    if (op->smem > 48 * 1024 &&
        cudaFuncSetAttribute(reinterpret_cast<const void*>(op->kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamicSmem) != cudaSuccess) {
      cudaGetLastError(); delete op; return fail("cannot raise the dynamic shared memory limit");
    }
  } else {
    const int mn = d->tile_rows;
    if ((mn != 32 && mn != 64) || d->splits < 1 || d->splits > 8 || d->splits > p.k_tiles) {
      delete op; return fail("bad tile form");
    }
    p.splits = d->splits;
    op->tile = d->dtype == kBF16 ? pick_tile<true>(sg, mn) : pick_tile<false>(sg, mn);
    op->grid = dim3((d->n + 127) / 128, (d->m + mn - 1) / mn, d->splits);
    const int stage = (2 * mn * 128 + static_cast<int>(p.block_bytes) + 1023) / 1024 * 1024;
    p.wide = wide; p.stage_bytes = static_cast<uint32_t>(stage);
    p.stages = std::min(kMaxInt4Stages, (227 * 1024 - 1024 - 1024) / stage);
    op->smem = p.stages * stage + 1024;
    EncodeTiledFn enc = get_encode_tiled();
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(d->k), static_cast<cuuint64_t>(d->m)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.x_ld) * 2};
    const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(mn)}, ones[2] = {1, 1};
    if (enc == nullptr ||
        enc(&op->tm_x, d->dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
            const_cast<uint8_t*>(p.x), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
      delete op; return fail("tensor map encoding failed");
    }
    if (cudaFuncSetAttribute(reinterpret_cast<const void*>(op->tile), cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamicSmem) != cudaSuccess) {
      cudaGetLastError(); delete op; return fail("cannot raise the dynamic shared memory limit");
    }
  }
  if (op->grid.y > 65535) { delete op; return fail("too many rows"); }
  return op;
}
