// Attention of a generating text model: whole prompts (causal or not, grouped heads, packed sequences of any length)
// and one new token per batch item over a prefix that the batch shares plus the item's own keys.
//
// With G = H / Hk query heads per key head, row r of a 128-row query tile is (token r / G, head r % G of the group), so
// one tile meets every K / V row of its key head once for all G heads. Per row, over its visible keys j:
//
//   s_j = scale * q . k_j      m = max_j s_j      l = sum_j 2^((s_j - m) log2 e)      o = sum_j 2^(...) v_j / l
//
// kept as a running (m, l, o) while K / V go by in tiles of 128 keys. tile_attention_kernel (tcgen05): a CTA owns two
// query tiles; one thread feeds TMA, one issues the MMAs, and four warps per query tile do the softmax, a thread per row:
//
//   S = Q K^T   (operands in shared memory, fp32 accumulator in tensor memory)
//   P = 2^(...) rounded to the inputs' 16-bit type and written over S in tensor memory (the A operand of the next MMA;
//               the row sum l is taken from the unrounded fp32 values, so P's rounding is the only one between the inputs
//               and the output's own: half a step of the 16-bit type each, 2^-8 (bf16) or 2^-11 of the weight, because the
//               tensor cores multiply 16-bit operands; P in two 16-bit parts would double the second product)
//   O += P V    (V as it lies in memory, keys by head columns: an MN-major operand, no transpose)
//
// The maximum a row is scaled by only moves when it grew by more than 8 in log2 units: until then p <= 2^8, which the
// 16-bit types and the fp32 sums hold without loss, and O needs no rescaling. fp16 has fixed steps of 2^-24 below 2^-14,
// which would take small weights away that together count (32768 weights of 2^-25 were lost to the last one), so fp16 weights
// are held 2^7 times as large (at most 2^15): below 2^-21 a weight is off by at most 2^-32, all of up to 2^20 keys together by
// 2^-12 of the largest. l and O carry the same factor, which the quotient does not see.
//
// One 16384-token causal sequence, 16 query heads over 4 of 128 columns, bf16: 1070 us, 1.03 PFLOP/s (1.4 is what a long
// cuBLAS product sustains). A pair of tiles takes 3700 clocks a key tile where the products need 2048 and the exponential
// unit 2048 (either pipe 55 % busy): what is left is the chain S -> maximum -> exponentials -> P of one tile, which only the
// other tile overlaps. A quarter of the exponentials as a polynomial on the FMA pipe was slower (1109 us: spilled registers).
// Short sequences are bound by a CTA's start and end (64 of 16 to 512 tokens, 12 heads of 64: 82 us, 13600 clocks a CTA with
// every pipe under 20 %).
//
// own_keys_kernel: an item's own keys are met by its G query rows alone, so that part is bound by the bytes of K and V;
// it brings them through a cp.async ring to the fragments of mma.sync and joins the two parts. 64 items, 4096 shared and 1
// to 512 own keys, 8 key heads of 128: 40 us, 128 items, 32768 shared and 64 to 1024 own keys: 157 us (the prefix 80, the own
// keys 72 at 3.9 TB/s).
//
// Every wait is bounded and reports through the status word.
#include "fdb_common.h"
#include "sm100_ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace fdb {

// Descriptor shared with ops/decoder.py.
struct DecoderAttnDesc {
  const void* q; const void* k; const void* v; void* out; int* status;   // prompt: q / k / v / out rows are tokens
  const int* seq_start; const int* seq_len;      // device int32, one per sequence (prefix form: seq_len per item)
  const void* pk; const void* pv;                // prefix rows (prefix form), may be null when prefix_rows is 0
  const int* prefix_len;                         // device int32 [1] or null: all prefix_rows
  void* part_o; void* part_ml; void* own_o; void* own_ml; unsigned* counter;     // workspaces of the prefix form
  long long q_ld, k_ld, v_ld, o_ld, pk_ld, pv_ld;        // row pitches in elements
  long long k_item, v_item;                      // prefix form: pitch between items of k / v, in elements
  int dtype, prefix_form;
  int n_seq, rows, max_len;                      // prompt: sequences, rows of the buffers, longest sequence
  int prefix_rows, own_rows;                     // prefix form: capacity of the prefix / of an item's own keys
  int H, Hk, D, causal, splits, own_splits;
  float scale;
};

struct TileParams {
  uint8_t* out; int* status;
  const int* seq_start; const int* seq_len; const int* prefix_len;
  float* part_o; float2* part_ml;
  long long o_ld;
  int n_seq, rows, max_len;
  int H, Hk, G, D, tok;          // tok = 128 / G: tokens of one query tile
  int causal, splits, tiles;     // prefix form: splits of the keys, pairs of query tiles
  int d_chunks, d_steps_last, stages, units;
  uint32_t q_box_bytes;          // bytes of one Q chunk that TMA writes
  float sl2;                     // scale * log2 e
};

constexpr int kTileThreads = 384;      // warps 0-3: query tile 0, warps 4-7: query tile 1, 8: MMA, 9: TMA, 10 and 11 idle
// Registers: 384 threads are launched with 168 each; the softmax warpgroups take 216 (a row's 128 scores stay in
// registers between the maximum and the exponentials), the third keeps 72: 128 * (2 * 216 + 72) = 384 * 168.
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
constexpr int kMaxStages = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleAbove = 8.f;   // log2 units
// log2 of the factor that 16-bit weights are held with (bf16 has fp32's range and needs none): for p <= 2^8, and for the own
// keys, whose maximum never lags, for p <= 1.
template <bool BF16> constexpr float kTileUp = BF16 ? 0.f : 7.f;
template <bool BF16> constexpr float kOwnUp = BF16 ? 0.f : 15.f;

__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if (BF16) { __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t*>(&h); }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two fp32 at a time, in one 64-bit register pair.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void of_pair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// What one CTA works on.
struct Unit {
  int q_row;          // first row of the sequence in q / out (prefix form: 0)
  int q_len;          // tokens of the sequence (prefix form: batch items)
  int k_row;          // first key row
  int k_len;          // keys of the sequence (prefix form: of the prefix)
  int tok0;           // first token of query tile 0
  int tile0;          // first key tile
  int n0, n1;         // key tiles of the two query tiles
  int head;           // key head
  int split;
};

template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <bool BF16, bool PREFIX>
__global__ void __launch_bounds__(kTileThreads, 1)
tile_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const TileParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 10];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ Unit unit;
  volatile int* abort_flag = &abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (PREFIX) launch_dependents();
  // ------------------------------------------------------------------------------------------ which unit is this CTA's
  if (warp == 0) {
    const int head = static_cast<int>(blockIdx.x) % p.Hk, want = static_cast<int>(blockIdx.x) / p.Hk;
    Unit u{};
    u.head = head;
    bool found = false;
    int bad = 0;
    if (PREFIX) {
      u.q_len = p.rows;
      u.k_len = p.max_len;
      if (p.prefix_len != nullptr) {
        const int n = __ldg(p.prefix_len);
        if (n < 0 || n > p.max_len) bad = 1;
        u.k_len = max(0, min(n, p.max_len));
      }
      u.split = want % p.splits;
      u.tok0 = want / p.splits * 2 * p.tok;
      const int all = (u.k_len + 127) / 128;
      u.tile0 = static_cast<int>(static_cast<long long>(all) * u.split / p.splits);
      const int n = static_cast<int>(static_cast<long long>(all) * (u.split + 1) / p.splits) - u.tile0;
      u.n0 = n;
      u.n1 = u.tok0 + p.tok < u.q_len ? n : 0;
      found = true;
    } else {
      int base = 0;
      for (int s0 = 0; s0 < p.n_seq && (!found || blockIdx.x == 0); s0 += 32) {
        const int s = s0 + lane;
        int st = 0, len = 0;
        if (s < p.n_seq) {
          st = __ldg(p.seq_start + s);
          len = __ldg(p.seq_len + s);
          if (len < 0 || len > p.max_len || st < 0 || st > p.rows - len) { bad |= len != 0; len = 0; }
        }
        const int t = (len + 2 * p.tok - 1) / (2 * p.tok);
        int incl = t;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) { const int x = __shfl_up_sync(0xffffffffu, incl, o); if (lane >= o) incl += x; }
        const unsigned hit = __ballot_sync(0xffffffffu, want < base + incl);
        if (!found && hit != 0) {
          const int from = __ffs(hit) - 1;
          const int idx = want - base - __shfl_sync(0xffffffffu, incl - t, from);
          const int tiles = __shfl_sync(0xffffffffu, t, from);
          u.q_len = u.k_len = __shfl_sync(0xffffffffu, len, from);
          u.q_row = u.k_row = __shfl_sync(0xffffffffu, st, from);
          u.tok0 = (p.causal ? tiles - 1 - idx : idx) * 2 * p.tok;      // the tiles with most keys first
          found = true;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (blockIdx.x == 0 && base > p.units) bad = 1;        // overlapping sequences: more tiles than the plan has CTAs
      auto tiles_of = [&](int first) {
        const int keys = p.causal ? min(u.k_len, first + p.tok) : u.k_len;
        return found && first < u.q_len ? (keys + 127) / 128 : 0;
      };
      u.n0 = tiles_of(u.tok0);
      u.n1 = tiles_of(u.tok0 + p.tok);
    }
    bad = __any_sync(0xffffffffu, bad);
    if (lane == 0) {
      unit = u;
      abort_word = 0;
      if (bad && p.status != nullptr) atomicCAS(p.status, 0, kStatusBadShape);
    }
  }
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t chunk = 16384u;                                   // 128 rows x 128 bytes
  const uint32_t q_tile_bytes = static_cast<uint32_t>(p.d_chunks) * chunk, stage_bytes = q_tile_bytes;
  const uint32_t s_q = base, s_ring = base + 2 * q_tile_bytes;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };
  // 0..7 full, 8..15 empty, then:
  const uint32_t bar_q = bar(16), bar_tail = bar(17);
  auto bar_s = [&](int t) { return bar(18 + t); };
  auto bar_o = [&](int t) { return bar(20 + t); };
  auto bar_p = [&](int t, int half) { return bar(22 + 2 * t + half); };        // 64 keys each
  if (warp == 9 && lane == 0) {
    for (int i = 0; i < kMaxStages; ++i) { mbar_init(bar(i), 1); mbar_init(bar(8 + i), 1); }
    mbar_init(bar_q, 1); mbar_init(bar_tail, 1);
    for (int t = 0; t < 2; ++t) { mbar_init(bar_s(t), 1); mbar_init(bar_o(t), 1); mbar_init(bar_p(t, 0), 4); mbar_init(bar_p(t, 1), 4); }
    fence_mbar_init();
    prefetch_tensormap(&tm_q); prefetch_tensormap(&tm_k); prefetch_tensormap(&tm_v);
  }
  __syncthreads();
  const Unit u = unit;
  const int n_all = max(u.n0, u.n1);
  auto n_of = [&](int t) { return t == 0 ? u.n0 : u.n1; };
  if (n_all == 0) {
    // nothing to do: an empty split of the prefix still says so
    if (PREFIX && p.part_ml != nullptr) {
      for (int r = tid; r < 2 * p.tok * p.G; r += kTileThreads) {
        const int item = u.tok0 + r / p.G;
        if (item < u.q_len)
          p.part_ml[(static_cast<long long>(u.split) * p.rows + item) * p.H + u.head * p.G + r % p.G] = make_float2(-INFINITY, 0.f);
      }
    }
    return;
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // last key (exclusive, counted from the unit's first key tile) that any row of query tile t sees
  auto key_end = [&](int t) {
    const int keys = p.causal ? min(u.k_len, u.tok0 + (t + 1) * p.tok) : u.k_len;
    return min(keys - u.tile0 * 128, n_of(t) * 128);
  };
  const int end_all = max(u.n0 > 0 ? key_end(0) : 0, u.n1 > 0 ? key_end(1) : 0);

  if (warp >= 8) {
  regs_dec<kOtherRegs>();
  if (warp == 9) {
    // ---------------------------------------------------------------------------------------------- TMA: Q, then K, V
    int issued = 0;
    auto load = [&](const CUtensorMap* tm, int row, uint32_t b, int st) {
      mbar_arrive_expect_tx(b, stage_bytes);
      for (int c = 0; c < p.d_chunks; ++c)
        tma_load_3d(s_ring + static_cast<uint32_t>(st) * stage_bytes + c * chunk, tm, b, c * 64, u.head, row);
    };
    if (lane == 0) {
      mbar_arrive_expect_tx(bar_q, static_cast<uint32_t>(p.d_chunks) * p.q_box_bytes * (u.n1 > 0 ? 2u : 1u));
      for (int t = 0; t < (u.n1 > 0 ? 2 : 1); ++t)
        for (int c = 0; c < p.d_chunks; ++c)
          tma_load_4d(s_q + t * q_tile_bytes + c * chunk, &tm_q, bar_q, c * 64, 0, u.head, u.q_row + u.tok0 + t * p.tok);
    }
    bool ok = true;
    RingAt at_ring{0, 0u};
    for (int i = 0; ok && i < 2 * n_all; ++i, at_ring.step(1, p.stages)) {
      const int st = at_ring.st;
      if (i >= p.stages) ok = mbar_wait_warp(bar(8 + st), at_ring.parity ^ 1u, abort_flag, kStatusTimeoutProducer);
      if (!ok) break;
      const int j = i >> 1, row = u.k_row + (u.tile0 + j) * 128;
      const int keys = end_all - j * 128;
      if ((i & 1) == 0) {
        if (lane == 0) load(&tm_k, row, bar(st), st);
      } else if (keys >= 128 || keys % 16 == 0) {
        if (lane == 0) load(&tm_v, row, bar(st), st);
      } else {
        // The last V tile ends inside a 16-key step: the rows behind it belong to something else and meet weights of
        // zero, but zero times an infinity is not zero. They are overwritten with zeros before the MMA may read them.
        if (lane == 0) load(&tm_v, row, bar_tail, st);
        __syncwarp();
        ok = mbar_wait_warp(bar_tail, 0, abort_flag, kStatusTimeoutProducer);
        const int pad = 16 - keys % 16;
        const uint32_t at = s_ring + static_cast<uint32_t>(st) * stage_bytes + static_cast<uint32_t>(keys) * 128u;
        for (int w = lane; ok && w < pad * 8 * p.d_chunks; w += 32) {
          const int c = w / (pad * 8), off = w % (pad * 8);
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + c * chunk + static_cast<uint32_t>(off) * 16u), "r"(0u) : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(st));
      }
      issued = i + 1;
    }
    // a CTA that gives up leaves no copy of its own in flight
    if (!ok && lane == 0) {
      volatile int none = 0;
      mbar_wait(bar_q, 0, &none, kStatusTimeoutProducer);
      for (int i = max(0, issued - p.stages); i < issued; ++i) {
        none = 0;
        mbar_wait(bar(i % p.stages), (i / p.stages) & 1, &none, kStatusTimeoutProducer);
      }
    }
    __syncwarp();
  } else if (warp == 8) {
    // ------------------------------------------------------------------------------------------------------------ MMA
    // one elected thread: the compiler then keeps descriptors in uniform registers
    if (elect_one()) {
      const uint32_t fmt = BF16 ? 1u : 0u;
      const uint32_t idesc_o = make_idesc(fmt, 128, static_cast<uint32_t>((p.D + 15) / 16 * 16)) | kIdescBMnMajor;
      auto qk = [&](int t, int j, int st) {
        const int keys = min(128, key_end(t) - j * 128);
        const uint32_t idesc = make_idesc(fmt, 128, static_cast<uint32_t>((keys + 15) / 16 * 16));
        const uint32_t sk = s_ring + static_cast<uint32_t>(st) * stage_bytes;
        for (int c = 0; c < p.d_chunks; ++c)
          umma_f16_ksteps(tmem + t * 128, make_kmajor_desc(s_q + t * q_tile_bytes + c * chunk, 128),
                          make_kmajor_desc(sk + c * chunk, 128), idesc, c != 0 ? 1u : 0u,
                          c + 1 == p.d_chunks ? static_cast<uint32_t>(p.d_steps_last) : 4u);
        umma_commit(bar_s(t));
      };
      auto pv = [&](int t, int j, int st) {
        const int keys = min(128, key_end(t) - j * 128);
        const uint64_t bd = make_mnmajor_desc(s_ring + static_cast<uint32_t>(st) * stage_bytes, chunk);
        const int steps = (keys + 15) / 16;
        // the second half of P is still being computed while the first one is multiplied
        for (int half = 0; half < 2; ++half) {
          if (!mbar_wait(bar_p(t, half), j & 1, abort_flag, kStatusTimeoutMma)) return false;
          tc_fence_after();
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int s = half * 4 + x;
            if (s < steps)
              umma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + s * 8, bd + static_cast<uint64_t>(s * 128), idesc_o,
                          (j | s) != 0 ? 1u : 0u);
          }
        }
        umma_commit(bar_o(t));
        return true;
      };
      bool ok = mbar_wait(bar_q, 0, abort_flag, kStatusTimeoutMma) && mbar_wait(bar(0), 0, abort_flag, kStatusTimeoutMma);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < 2; ++t) if (n_of(t) > 0) qk(t, 0, 0);
        umma_commit(bar(8));
      }
      RingAt at_v{1, 0u};                                            // K_0 V_0 K_1 V_1 ... in the ring (three stages or more)
      for (int j = 0; ok && j < n_all; ++j) {
        RingAt at_k = at_v;
        at_k.step(1, p.stages);
        ok = mbar_wait(bar(at_v.st), at_v.parity, abort_flag, kStatusTimeoutMma);
        if (ok && j + 1 < n_all) ok = mbar_wait(bar(at_k.st), at_k.parity, abort_flag, kStatusTimeoutMma);
        for (int t = 0; ok && t < 2; ++t) {
          if (j >= n_of(t)) continue;
          ok = pv(t, j, at_v.st);
          if (!ok) break;
          if (j + 1 < n_of(t)) qk(t, j + 1, at_k.st);
        }
        if (ok) {
          umma_commit(bar(8 + at_v.st));
          if (j + 1 < n_all) umma_commit(bar(8 + at_k.st));
        }
        at_v = at_k;
        at_v.step(1, p.stages);
      }
    }
    __syncwarp();
  }
  } else {
    regs_inc<kSoftmaxRegs>();
    // ---------------------------------------------------------------------------------------------- softmax, a row each
    const int t = warp >> 2, r = tid & 127, n = n_of(t);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + t * 128 + lanes, t_o = tmem + 256 + t * 128 + lanes;
    const int first = u.tok0 + t * p.tok;
    const int token = first + r / p.G;
    const bool real = r < p.tok * p.G && token < u.q_len;
    const int end = n > 0 ? key_end(t) : 0;
    // keys of the unit that this row sees; rows that are no query keep the tile's bound
    const int row_end = p.causal ? min(end, token + 1 - u.tile0 * 128) : end;
    const int full_end = p.causal ? min(end, first + 1 - u.tile0 * 128) : end;     // every row of the tile sees these
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; ok && j < n; ++j) {
      ok = mbar_wait(bar_s(t), j & 1, abort_flag, kStatusTimeoutMma);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int blocks = (min(128, end - j * 128) + 31) / 32;
      const bool full = (j + 1) * 128 <= full_end;
      const int lim = row_end - j * 128;
      uint32_t v[4][32];
      float m_new = m;
      // the next 32 columns are on their way out of tensor memory while these are compared
      tmem_ld_32x32(t_s, v[0]);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        if (b >= blocks) continue;
        tmem_ld_wait_dep(v[b]);
        if (b < 3 && b + 1 < blocks) tmem_ld_32x32(t_s + (b + 1) * 32, v[(b + 1) & 3]);
        if (!full) {
#pragma unroll
          for (int c = 0; c < 32; ++c) if (b * 32 + c >= lim) v[b][c] = 0xff800000u;      // minus infinity
        }
        float m4[4] = {m_new, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 32; c += 2)
          m4[(c >> 1) & 3] = max3(m4[(c >> 1) & 3], __uint_as_float(v[b][c]), __uint_as_float(v[b][c + 1]));
        m_new = max3(fmaxf(m4[0], m4[1]), m4[2], m4[3]);
      }
      const bool grow = m != -INFINITY && (m_new - m) * p.sl2 > kRescaleAbove;
      if (m == -INFINITY) m = m_new;
      if (__any_sync(0xffffffffu, grow)) {
        float a = 1.f;
        if (grow) { a = exp2_ftz((m - m_new) * p.sl2); m = m_new; l *= a; }
        ok = mbar_wait(bar_o(t), (j - 1) & 1, abort_flag, kStatusTimeoutMma);     // O of the tiles so far is complete
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        for (int c0 = 0; c0 < p.D; c0 += 32) {
          uint32_t o[32];
          tmem_ld_32x32(t_o + c0, o);
          tmem_ld_wait_dep(o);
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * a);
          tmem_st_32x32(t_o + c0, o);
        }
        tmem_st_wait();
      }
      const float off = m == -INFINITY ? 0.f : kTileUp<BF16> - m * p.sl2;
      const uint64_t scale2 = pair_of(p.sl2, p.sl2), off2 = pair_of(off, off);
      uint64_t sum2[2] = {0, 0};                                     // zeros
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (2 * h < blocks) {
          uint32_t w[32];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            if (2 * h + b < blocks) {
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                float e0, e1;
                of_pair(fma2(pair_of(__uint_as_float(v[2 * h + b][2 * c]), __uint_as_float(v[2 * h + b][2 * c + 1])), scale2, off2), e0, e1);
                e0 = exp2_ftz(e0);
                e1 = exp2_ftz(e1);
                sum2[c & 1] = add2(sum2[c & 1], pair_of(e0, e1));
                w[b * 16 + c] = pack_pair<BF16>(e0, e1);
              }
            } else {
#pragma unroll
              for (int c = 0; c < 16; ++c) w[b * 16 + c] = 0u;
            }
          }
          tmem_st_32x32(t_s + h * 32, w);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p(t, h));
      }
      float e0, e1;
      of_pair(add2(sum2[0], sum2[1]), e0, e1);
      l += e0 + e1;
    }
    if (ok && n > 0) {
      ok = mbar_wait(bar_o(t), (n - 1) & 1, abort_flag, kStatusTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok && n > 0) {
      tc_fence_after();
      // A thread owns a row, and rows are far apart in memory: stored from here, a warp's instruction would touch 32 lines
      // (the fp32 parts of 256 rows of 128 took 9000 clocks). So a warp turns its 32 rows, 128 bytes of each at a time,
      // around in the shared memory of this tile's queries, which the finished MMAs no longer read: eight threads then
      // write a row's 128 bytes. Pieces of 16 bytes are permuted by the row, both ways without bank conflicts.
      const int head = u.head * p.G + r % p.G;
      uint8_t* mine = nullptr;
      if (real) {
        const long long row = (static_cast<long long>(u.split) * p.rows + token) * p.H + head;
        if (PREFIX) p.part_ml[row] = make_float2(m == -INFINITY ? m : m * p.sl2 - kTileUp<BF16>, l);
        mine = PREFIX ? reinterpret_cast<uint8_t*>(p.part_o + row * p.D)
                      : p.out + ((static_cast<long long>(u.q_row) + token) * p.o_ld + static_cast<long long>(head) * p.D) * 2;
      }
      const float inv = PREFIX ? 1.f : 1.f / l;
      const uint32_t turn = s_q + t * q_tile_bytes + static_cast<uint32_t>(warp & 3) * 4096u;
      constexpr int kCols = PREFIX ? 32 : 64;                        // columns of O in 128 bytes
      const int row_bytes = p.D * (PREFIX ? 4 : 2);
      for (int c0 = 0; c0 < p.D; c0 += kCols) {
        uint32_t w[32];
        if (PREFIX) {
          tmem_ld_32x32(t_o + c0, w);
          tmem_ld_wait_dep(w);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t o[32];
            tmem_ld_32x32(t_o + c0 + h * 32, o);
            tmem_ld_wait_dep(o);
#pragma unroll
            for (int c = 0; c < 16; ++c)
              w[h * 16 + c] = pack_pair<BF16>(__uint_as_float(o[2 * c]) * inv, __uint_as_float(o[2 * c + 1]) * inv);
          }
        }
        __syncwarp();                                                // the last 128 bytes have been read
#pragma unroll
        for (int c = 0; c < 8; ++c)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(turn + lane * 128 + ((c ^ (lane & 7)) << 4)),
                       "r"(w[4 * c]), "r"(w[4 * c + 1]), "r"(w[4 * c + 2]), "r"(w[4 * c + 3]) : "memory");
        __syncwarp();
        const int at = c0 * (PREFIX ? 4 : 2) + (lane & 7) * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int from = i * 4 + (lane >> 3);
          uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), from));
          uint4 x;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                       : "r"(turn + from * 128 + (((lane & 7) ^ (from & 7)) << 4)) : "memory");
          if (to != nullptr && at < row_bytes) *reinterpret_cast<uint4*>(to + at) = x;
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (tid == 0 && abort_word != 0 && p.status != nullptr) atomicCAS(p.status, 0, abort_word);
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// ------------------------------------------------------------------------------------------------- an item's own keys
struct OwnParams {
  const uint8_t* q; const uint8_t* k; const uint8_t* v; uint8_t* out; int* status;
  const int* seq_len; const int* prefix_len;
  const float* part_o; const float2* part_ml;        // the prefix's parts [splits][B][H](D)
  float* own_o; float2* own_ml; unsigned* counter;   // own parts [own_splits][B][H](D), one counter per (item, CTA column)
  long long q_ld, k_ld, v_ld, o_ld, k_item, v_item;
  int B, H, Hk, G, D, own_rows, prefix_rows, splits, own_splits, columns;   // columns = CTAs per item (key heads x head chunks)
  float sl2;
};

constexpr int kOwnWarps = 4;

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                            uint32_t b1, bool bf16) {
  if (bf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// One CTA: one item, one key head, up to 8 NT of its query heads, one split of the item's own keys. A warp takes 16 keys
// at a time, which it brings into a ring of its own in shared memory by cp.async, two tiles ahead (16 KB a warp in flight
// for 128 columns). Scores come transposed,
// S^T [16 keys x heads] = K Q^T, so that K rows are the A operand as 16-byte reads deliver them (the order of the head
// columns inside an MMA is free as long as Q follows it), and O^T [head columns x heads] = V^T P takes V rows the same way
// after pairing two keys' halves with prmt. Pieces of 16 bytes are permuted within a row by a function of the row, so that
// both kinds of reads meet all banks.
constexpr int kOwnStages = 3;

__host__ __device__ constexpr int own_stage_bytes(int dp) { return 2 * 16 * dp * 2; }
inline int own_smem_bytes(int dp, int nt, int parts) {
  const int ring = kOwnWarps * kOwnStages * own_stage_bytes(dp);
  const int join = (kOwnWarps * 8 * nt * dp + 2 * 8 * nt * (parts + kOwnWarps)) * 4;
  return std::max(ring, join);
}

template <bool BF16, int DP, int NT>
__global__ void __launch_bounds__(kOwnWarps * 32)
own_keys_kernel(const OwnParams p) {
  constexpr int KC = DP / 32, VC = DP / 64, kRow = DP * 2, kUnits = DP / 8, kRowsAtOnce = 32 / kUnits;
  extern __shared__ __align__(16) uint8_t own_smem[];
  __shared__ float2 sm_ml[kOwnWarps][8 * NT];
  __shared__ float sm_inv[8 * NT];
  __shared__ unsigned ticket;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int column = blockIdx.x % p.columns, item = blockIdx.x / p.columns;
  const int chunks = p.columns / p.Hk, hk = column / chunks, h0 = column % chunks * (8 * NT);
  const int heads = min(8 * NT, p.G - h0);                          // query heads of this CTA
  const int head0 = hk * p.G + h0;
  uint4 q[NT][KC];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int h = i * 8 + g, d = c * 32 + t * 8;
      q[i][c] = make_uint4(0, 0, 0, 0);
      if (h < heads && d < p.D)
        q[i][c] = __ldg(reinterpret_cast<const uint4*>(p.q + (item * p.q_ld + static_cast<long long>(head0 + h) * p.D + d) * 2));
    }
  int len = p.own_rows;
  if (p.own_rows > 0) {
    const int n = __ldg(p.seq_len + item);
    if ((n < 0 || n > p.own_rows) && threadIdx.x == 0 && p.status != nullptr) atomicCAS(p.status, 0, kStatusBadShape);
    len = max(0, min(n, p.own_rows));
  }
  const int per = (((len + p.own_splits - 1) / p.own_splits) + 15) / 16 * 16;
  const int k0 = min(len, static_cast<int>(blockIdx.y) * per), k1 = min(len, k0 + per);

  // ---- the warp's ring: tile i is keys k0 + (warp + kOwnWarps i) * 16 .. of K and of V
  const uint8_t* ring = own_smem + warp * (kOwnStages * own_stage_bytes(DP));
  const uint32_t ring_at = smem_u32(ring);
  const uint8_t* kb = p.k + (item * p.k_item + static_cast<long long>(hk) * p.D) * 2;
  const uint8_t* vb = p.v + (item * p.v_item + static_cast<long long>(hk) * p.D) * 2;
  const int unit = lane % kUnits, row0 = lane / kUnits;
  const bool unit_in = unit * 8 < p.D;
  auto swizzle = [](int row) { return (((row >> 1) & 3) * 2) ^ ((row & 1) * 4); };
  auto fetch = [&](int key, int stage) {
    if (key < k1) {
      const uint32_t at = ring_at + static_cast<uint32_t>(stage) * own_stage_bytes(DP);
#pragma unroll
      for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
        const int row = row0 + i * kRowsAtOnce;
        const bool in = unit_in && key + row < k1;                  // what is not read is filled with zeros
        const uint32_t to = at + row * kRow + (((unit & ~7) | ((unit & 7) ^ swizzle(row))) * 16);
        cp_async_16(to, in ? kb + ((key + row) * p.k_ld + unit * 8) * 2 : kb, in ? 16 : 0);
        cp_async_16(to + 16 * kRow, in ? vb + ((key + row) * p.v_ld + unit * 8) * 2 : vb, in ? 16 : 0);
      }
    }
    cp_async_commit();
  };
  const int first = k0 + warp * 16;
#pragma unroll
  for (int i = 0; i < kOwnStages - 1; ++i) fetch(first + i * kOwnWarps * 16, i);

  float o[NT][2 * VC][2][4] = {};       // [heads][64-column half: 4 m16 tiles as 2 x 2][..]: see the store below
  float mx[NT][2], sum[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) { mx[i][0] = mx[i][1] = -INFINITY; sum[i][0] = sum[i][1] = 0.f; }

  int stage = 0;
  for (int key = first; key < k1; key += kOwnWarps * 16) {
    cp_async_wait<kOwnStages - 2>();
    __syncwarp();                                                   // every lane's copies of this tile have landed
    const int free_stage = stage == 0 ? kOwnStages - 1 : stage - 1; // the one that the previous tile left
    fetch(key + (kOwnStages - 1) * kOwnWarps * 16, free_stage);
    const uint8_t* at = ring + stage * own_stage_bytes(DP);
    stage = stage + 1 == kOwnStages ? 0 : stage + 1;
    float s[NT][4] = {};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      const int u = c * 4 + t, x = (u & ~7) | ((u & 7) ^ swizzle(g));
      const uint4 ka = *reinterpret_cast<const uint4*>(at + g * kRow + x * 16);
      const uint4 kc = *reinterpret_cast<const uint4*>(at + (g + 8) * kRow + x * 16);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        mma_16x8x16(s[i], ka.x, kc.x, ka.y, kc.y, q[i][c].x, q[i][c].y, BF16);
        mma_16x8x16(s[i], ka.z, kc.z, ka.w, kc.w, q[i][c].z, q[i][c].w, BF16);
      }
    }
    // s[0], s[1]: key g, heads 2t and 2t + 1; s[2], s[3]: key g + 8
    const bool in0 = key + g < k1, in1 = key + g + 8 < k1;
    float a[NT][2];
    uint32_t b0[NT], b1[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float e[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float s0 = in0 ? s[i][x] * p.sl2 : -INFINITY, s1 = in1 ? s[i][2 + x] * p.sl2 : -INFINITY;
        float w = fmaxf(s0, s1);
        w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 4));
        w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 8));
        w = fmaxf(w, __shfl_xor_sync(0xffffffffu, w, 16));
        w = fmaxf(w, mx[i][x]);
        const float top = w == -INFINITY ? 0.f : w, base = top - kOwnUp<BF16>;
        a[i][x] = exp2_ftz(mx[i][x] - top);
        mx[i][x] = w;
        e[x] = exp2_ftz(s0 - base);
        e[2 + x] = exp2_ftz(s1 - base);
        sum[i][x] = sum[i][x] * a[i][x] + e[x] + e[2 + x];
      }
      b0[i] = transpose_8x8(pack_pair<BF16>(e[0], e[1]));
      b1[i] = transpose_8x8(pack_pair<BF16>(e[2], e[3]));
    }
#pragma unroll
    for (int c = 0; c < VC; ++c) {
      uint4 vv[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = 2 * t + (x & 1) + (x >> 1) * 8;
        vv[x] = *reinterpret_cast<const uint4*>(at + 16 * kRow + row * kRow + (c * 8 + (g ^ swizzle(row))) * 16);
      }
      const uint32_t r0[4] = {vv[0].x, vv[0].y, vv[0].z, vv[0].w}, r1[4] = {vv[1].x, vv[1].y, vv[1].z, vv[1].w};
      const uint32_t r2[4] = {vv[2].x, vv[2].y, vv[2].z, vv[2].w}, r3[4] = {vv[3].x, vv[3].y, vv[3].z, vv[3].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t a0 = __byte_perm(r0[w], r1[w], 0x5410), a1 = __byte_perm(r0[w], r1[w], 0x7632);
        const uint32_t a2 = __byte_perm(r2[w], r3[w], 0x5410), a3 = __byte_perm(r2[w], r3[w], 0x7632);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float (&acc)[4] = o[i][2 * c + (w >> 1)][w & 1];
          acc[0] *= a[i][0]; acc[1] *= a[i][1]; acc[2] *= a[i][0]; acc[3] *= a[i][1];
          mma_16x8x16(acc, a0, a1, a2, a3, b0[i], b1[i], BF16);
        }
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();                                                  // the rings become the warps' parts
  float* sm_o = reinterpret_cast<float*>(own_smem);                 // [warp][head][column]
  float* sm_w = sm_o + kOwnWarps * 8 * NT * DP;                     // [head][part]: weights of the parts that are joined
  float* sm_l = sm_w + 8 * NT * (p.splits + (p.own_splits == 1 ? kOwnWarps : p.own_splits));     // their sums
#pragma unroll
  for (int i = 0; i < NT; ++i) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float w = sum[i][x];
      w += __shfl_xor_sync(0xffffffffu, w, 4);
      w += __shfl_xor_sync(0xffffffffu, w, 8);
      w += __shfl_xor_sync(0xffffffffu, w, 16);
      if (g == 0) sm_ml[warp][i * 8 + 2 * t + x] = make_float2(mx[i][x] - kOwnUp<BF16>, w);
    }
#pragma unroll
    for (int c = 0; c < VC; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          sm_o[(warp * 8 * NT + i * 8 + 2 * t + (x & 1)) * DP + c * 64 + g * 8 + 2 * w + (x >> 1)] = o[i][2 * c + (w >> 1)][w & 1][x];
  }
  __syncthreads();
  const int lanes_d = p.D / 4;                                      // a thread handles four columns of one head
  const bool single = p.own_splits == 1;
  if (!single) {
    for (int x = threadIdx.x; x < heads * lanes_d; x += blockDim.x) {
      const int h = x / lanes_d, d = x % lanes_d * 4;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kOwnWarps; ++w) m = fmaxf(m, sm_ml[w][h].x);
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kOwnWarps; ++w) {
        const float2 ml = sm_ml[w][h];
        if (ml.y == 0.f) continue;                                  // no keys (a NaN sum goes on)
        const float f = exp2_ftz(ml.x - m);
        const float4 v = *reinterpret_cast<const float4*>(&sm_o[(w * 8 * NT + h) * DP + d]);
        l += ml.y * f;
        r.x += v.x * f; r.y += v.y * f; r.z += v.z * f; r.w += v.w * f;
      }
      const long long row = (static_cast<long long>(blockIdx.y) * p.B + item) * p.H + head0 + h;
      *reinterpret_cast<float4*>(p.own_o + row * p.D + d) = r;
      if (d == 0) p.own_ml[row] = make_float2(m, l);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) ticket = atomicAdd(p.counter + blockIdx.x, 1u);
    __syncthreads();
    if (ticket != static_cast<unsigned>(p.own_splits) - 1u) return;
    if (threadIdx.x == 0) p.counter[blockIdx.x] = 0u;               // ready for the next launch
    __threadfence();
  }
  int prefix = p.prefix_rows;
  if (p.prefix_len != nullptr && prefix > 0) prefix = max(0, min(__ldg(p.prefix_len), prefix));
  const bool any_key = len > 0 || prefix > 0;
  wait_prerequisites();                                             // the prefix's parts
  // ---- join: parts 0 .. own - 1 are this item's own (this CTA's warps, or the splits), the rest the prefix's. First a
  // warp per head turns their maxima into weights, then each thread adds its columns of them, in order. A part without a
  // weight above zero (no keys, or none above minus infinity) gets the weight -1 and is left out: nobody may have written its
  // columns. All others take part whatever their weight: a NaN reaches the result though its part's maximum is small.
  const int own = single ? kOwnWarps : p.own_splits, parts = own + p.splits;
  auto part_row = [&](int s, int h) { return (static_cast<long long>(s) * p.B + item) * p.H + head0 + h; };
  for (int h = warp; h < heads; h += kOwnWarps) {
    auto stat = [&](int s) {
      if (s >= own) return __ldcg(p.part_ml + part_row(s - own, h));
      return single ? sm_ml[s][h] : __ldcg(p.own_ml + part_row(s, h));
    };
    float m = -INFINITY;
    for (int s = lane; s < parts; s += 32) {
      const float2 ml = stat(s);
      sm_w[h * parts + s] = ml.x;
      sm_l[h * parts + s] = ml.y;
      if (ml.y != 0.f) m = fmaxf(m, ml.x);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    float l = 0.f;
    for (int s = lane; s < parts; s += 32) {
      const float part_l = sm_l[h * parts + s];
      const float w = part_l == 0.f ? -1.f : exp2_ftz(sm_w[h * parts + s] - m);
      sm_w[h * parts + s] = w;
      if (part_l != 0.f) l += w * part_l;
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (lane == 0) sm_inv[h] = any_key ? 1.f / l : 0.f;             // no key at all: zeros
  }
  __syncthreads();
  for (int x = threadIdx.x; x < heads * lanes_d; x += blockDim.x) {
    const int h = x / lanes_d, d = x % lanes_d * 4;
    const float* weight = sm_w + h * parts;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (single) {
#pragma unroll
      for (int w = 0; w < kOwnWarps; ++w) {
        const float f = weight[w];
        const float4 v = *reinterpret_cast<const float4*>(&sm_o[(w * 8 * NT + h) * DP + d]);
        if (!(f < 0.f)) { r.x += v.x * f; r.y += v.y * f; r.z += v.z * f; r.w += v.w * f; }
      }
    }
    // eight parts' loads at a time are in flight
    auto add = [&](const float* src, long long pitch, const float* w, int n) {
      for (int s0 = 0; s0 < n; s0 += 8) {
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (s0 + k < n) v[k] = __ldcg(reinterpret_cast<const float4*>(src + (s0 + k) * pitch));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float f = s0 + k < n ? w[s0 + k] : -1.f;
          if (!(f < 0.f)) { r.x += v[k].x * f; r.y += v[k].y * f; r.z += v[k].z * f; r.w += v[k].w * f; }
        }
      }
    };
    const long long pitch = static_cast<long long>(p.B) * p.H * p.D, at = part_row(0, h) * p.D + d;
    if (!single) add(p.own_o + at, pitch, weight, own);
    add(p.part_o + at, pitch, weight + own, p.splits);
    const float inv = sm_inv[h];
    uint2 w;
    w.x = pack_pair<BF16>(r.x * inv, r.y * inv);
    w.y = pack_pair<BF16>(r.z * inv, r.w * inv);
    *reinterpret_cast<uint2*>(p.out + (item * p.o_ld + static_cast<long long>(head0 + h) * p.D + d) * 2) = w;
  }
}

}  // namespace fdb

using namespace fdb;

namespace {

bool encode(CUtensorMap* m, bool bf16, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
  EncodeTiledFn enc = get_encode_tiled();
  if (enc == nullptr) return false;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base),
             dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows [n][heads * D] with pitch ld as (D, heads, n), 128 rows of 64 columns of one head per box. Columns past D read as
// zeros, so a head size that is no multiple of 64 (or 16) never meets its neighbour's columns.
bool encode_kv(CUtensorMap* m, bool bf16, const void* base, int D, int heads, int rows, long long ld) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[3] = {64, 1, 128};
  return encode(m, bf16, base, 3, dims, strides, box);
}

// Query rows as (D, G, Hk, n): a box is `tok` rows of the G heads of one group.
bool encode_q(CUtensorMap* m, bool bf16, const void* base, int D, int G, int Hk, int rows, long long ld, int tok) {
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(G), static_cast<cuuint64_t>(Hk),
                              static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(G) * D * 2,
                                 static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(G), 1, static_cast<cuuint32_t>(tok)};
  return encode(m, bf16, base, 4, dims, strides, box);
}

struct DecoderAttnOp : Op {
  CUtensorMap tq, tk, tv;
  TileParams tile{};
  OwnParams own{};
  int device = 0, tile_grid = 0, smem = 0, own_smem = 0, nt = 1;
  dim3 own_grid;
  bool bf16 = true, prefix = false, wide = false;

  template <typename K, typename... A>
  cudaError_t dependent(K kernel, dim3 grid, int threads, cudaStream_t s, bool chained, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = own_smem; cfg.stream = s;
    if (chained) {
      at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at.val.programmaticStreamSerializationAllowed = 1;
      cfg.attrs = &at; cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
  }
  template <bool B>
  void (*own_kernel())(const OwnParams) {
    if (wide) return nt == 1 ? own_keys_kernel<B, 128, 1> : own_keys_kernel<B, 128, 2>;
    return nt == 1 ? own_keys_kernel<B, 64, 1> : own_keys_kernel<B, 64, 2>;
  }
  cudaError_t launch_own(cudaStream_t s) {
    return dependent(bf16 ? own_kernel<true>() : own_kernel<false>(), own_grid, kOwnWarps * 32, s, tile_grid > 0, own);
  }
  int launch(cudaStream_t s) override {
    int at = device;
    cudaGetDevice(&at);
    if (at != device) cudaSetDevice(device);
    if (tile_grid > 0) {
      if (prefix) {
        if (bf16) tile_attention_kernel<true, true><<<tile_grid, kTileThreads, smem, s>>>(tq, tk, tv, tile);
        else tile_attention_kernel<false, true><<<tile_grid, kTileThreads, smem, s>>>(tq, tk, tv, tile);
      } else {
        if (bf16) tile_attention_kernel<true, false><<<tile_grid, kTileThreads, smem, s>>>(tq, tk, tv, tile);
        else tile_attention_kernel<false, false><<<tile_grid, kTileThreads, smem, s>>>(tq, tk, tv, tile);
      }
    }
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && prefix) e = launch_own(s);
    if (at != device) cudaSetDevice(at);
    if (e != cudaSuccess) { set_error(std::string("decoder attention: ") + cudaGetErrorString(e)); return -1; }
    return 0;
  }
};

}  // namespace

FDB_API int fdb_decoder_attention_desc_size() { return static_cast<int>(sizeof(DecoderAttnDesc)); }

FDB_API void* fdb_decoder_attention_create(const DecoderAttnDesc* d) {
  auto fail = [](const std::string& what) -> void* { set_error("decoder attention: " + what); return nullptr; };
  if (d->dtype != kF16 && d->dtype != kBF16) return fail("dtype must be fp16 or bf16");
  if (!(d->scale > 0.f) || !(d->scale < INFINITY)) return fail("the score scale must be positive and finite");
  if (d->D < 8 || d->D > 128 || d->D % 8) return fail("the head dim must be a multiple of 8 in 8..128");
  if (d->H < 1 || d->Hk < 1 || d->H % d->Hk || d->H / d->Hk > 128) return fail("heads must be kv_heads times 1..128");
  auto al16 = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
  auto pitch = [](long long ld, long long least) { return ld % 8 == 0 && ld >= least; };
  const long long qw = static_cast<long long>(d->H) * d->D, kw = static_cast<long long>(d->Hk) * d->D;
  const bool pf = d->prefix_form != 0;
  const bool has_tile = !pf || d->prefix_rows > 0, has_own = pf && d->own_rows > 0;
  const void* tk = pf ? d->pk : d->k;
  const void* tv = pf ? d->pv : d->v;
  const long long tk_ld = pf ? d->pk_ld : d->k_ld, tv_ld = pf ? d->pv_ld : d->v_ld;
  const int t_rows = pf ? d->prefix_rows : d->rows;
  if (d->rows < 1 || d->prefix_rows < 0 || d->own_rows < 0) return fail("empty or negative sizes");
  if (!al16(d->q) || !al16(d->out) || !pitch(d->q_ld, qw) || !pitch(d->o_ld, qw))
    return fail("q and out must be 16-byte aligned with row pitches that are multiples of 8 elements and hold all heads");
  if (has_tile && (!al16(tk) || !al16(tv) || !pitch(tk_ld, kw) || !pitch(tv_ld, kw)))
    return fail("k and v must be 16-byte aligned with row pitches that are multiples of 8 elements and hold all heads");
  if (has_own && (!al16(d->k) || !al16(d->v) || !pitch(d->k_ld, kw) || !pitch(d->v_ld, kw) || d->k_item % 8 || d->v_item % 8 ||
                  d->seq_len == nullptr))
    return fail("the items' k and v must be 16-byte aligned with pitches that are multiples of 8 elements, with seq_len");
  if (!pf && (d->n_seq < 1 || d->max_len < 1 || d->seq_start == nullptr || d->seq_len == nullptr))
    return fail("a prompt needs seq_start, seq_len and max_len");

  auto* op = new DecoderAttnOp();
  cudaGetDevice(&op->device);
  op->bf16 = d->dtype == kBF16;
  op->prefix = pf;
  const int G = d->H / d->Hk;
  TileParams& t = op->tile;
  t.out = static_cast<uint8_t*>(d->out); t.status = d->status;
  t.seq_start = d->seq_start; t.seq_len = d->seq_len; t.prefix_len = d->prefix_len;
  t.part_o = static_cast<float*>(d->part_o); t.part_ml = static_cast<float2*>(d->part_ml);
  t.o_ld = d->o_ld;
  t.n_seq = d->n_seq; t.rows = d->rows; t.max_len = pf ? d->prefix_rows : std::min(d->max_len, d->rows);
  t.H = d->H; t.Hk = d->Hk; t.G = G; t.D = d->D; t.tok = 128 / G;
  t.causal = pf ? 0 : d->causal;
  t.splits = d->splits;
  t.d_chunks = (d->D + 63) / 64;
  t.d_steps_last = ((d->D - (t.d_chunks - 1) * 64) + 15) / 16;
  t.q_box_bytes = static_cast<uint32_t>(t.tok) * G * 128u;
  t.sl2 = d->scale * kLog2e;
  const int q_bytes = 2 * t.d_chunks * 16384, stage_bytes = t.d_chunks * 16384;
  t.stages = std::min(kMaxStages, (227 * 1024 - 2048 - 1024 - q_bytes) / stage_bytes);
  op->smem = q_bytes + t.stages * stage_bytes + 1024;
  if (has_tile) {
    const int pair = 2 * t.tok;
    long long units;
    if (pf) {
      if (d->splits < 1 || d->part_o == nullptr || d->part_ml == nullptr) { delete op; return fail("the prefix needs its workspace"); }
      t.tiles = (d->rows + pair - 1) / pair;
      units = static_cast<long long>(t.tiles) * d->splits;
    } else {
      // non-overlapping sequences: every one but for its last pair of tiles fills 2 * tok rows
      units = std::min(static_cast<long long>(d->rows / pair) + d->n_seq,
                       static_cast<long long>(d->n_seq) * ((t.max_len + pair - 1) / pair));
    }
    if (units * d->Hk > 0x7fffffffLL) { delete op; return fail("too many tiles for one launch"); }
    t.units = static_cast<int>(units);
    op->tile_grid = static_cast<int>(units * d->Hk);
    if (!encode_q(&op->tq, op->bf16, d->q, d->D, G, d->Hk, d->rows, d->q_ld, t.tok) ||
        !encode_kv(&op->tk, op->bf16, tk, d->D, d->Hk, t_rows, tk_ld) ||
        !encode_kv(&op->tv, op->bf16, tv, d->D, d->Hk, t_rows, tv_ld)) {
      delete op; return fail("tensor map encoding failed");
    }
    const void* fn = pf ? (op->bf16 ? reinterpret_cast<const void*>(&tile_attention_kernel<true, true>)
                                    : reinterpret_cast<const void*>(&tile_attention_kernel<false, true>))
                        : (op->bf16 ? reinterpret_cast<const void*>(&tile_attention_kernel<true, false>)
                                    : reinterpret_cast<const void*>(&tile_attention_kernel<false, false>));
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamicSmem) != cudaSuccess) {
      cudaGetLastError(); delete op; return fail("cannot raise the dynamic shared memory limit");
    }
  }
  if (pf) {
    OwnParams& o = op->own;
    o.q = static_cast<const uint8_t*>(d->q); o.k = static_cast<const uint8_t*>(d->k); o.v = static_cast<const uint8_t*>(d->v);
    o.out = static_cast<uint8_t*>(d->out); o.status = d->status; o.seq_len = d->seq_len; o.prefix_len = d->prefix_len;
    o.part_o = t.part_o; o.part_ml = t.part_ml;
    o.own_o = static_cast<float*>(d->own_o); o.own_ml = static_cast<float2*>(d->own_ml); o.counter = d->counter;
    o.q_ld = d->q_ld; o.k_ld = d->k_ld; o.v_ld = d->v_ld; o.o_ld = d->o_ld; o.k_item = d->k_item; o.v_item = d->v_item;
    o.B = d->rows; o.H = d->H; o.Hk = d->Hk; o.G = G; o.D = d->D; o.own_rows = d->own_rows; o.prefix_rows = d->prefix_rows;
    o.splits = has_tile ? d->splits : 0; o.own_splits = std::max(1, d->own_splits); o.sl2 = t.sl2;
    op->nt = G > 8 ? 2 : 1;
    op->wide = d->D > 64;
    o.columns = d->Hk * ((G + 8 * op->nt - 1) / (8 * op->nt));
    if (o.own_splits > 1 && (d->own_o == nullptr || d->own_ml == nullptr || d->counter == nullptr)) {
      delete op; return fail("split own keys need their workspace");
    }
    op->own_grid = dim3(static_cast<unsigned>(o.columns) * d->rows, o.own_splits);
    op->own_smem = own_smem_bytes(op->wide ? 128 : 64, op->nt, o.splits + o.own_splits);
    if (op->own_smem > kMaxDynamicSmem) { delete op; return fail("too many splits"); }
    const void* fn = reinterpret_cast<const void*>(op->bf16 ? op->own_kernel<true>() : op->own_kernel<false>());
    if (op->own_smem > 40 * 1024 && cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynamicSmem) != cudaSuccess) {
      cudaGetLastError(); delete op; return fail("cannot raise the dynamic shared memory limit");
    }
  }
  return op;
}
