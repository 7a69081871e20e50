// Projections with 4-bit weights and group scales for a few tokens (declarations: include/swiglu_b200.h):
//
//   y[m][n] = sum_k x[m][k] * (q[n][k] - z[n][k/G]) * s[n][k/G]            q in 0..15, G = 32, 64 or 128
//   h[m][n] = act(gm * (x . w_gate[n])) * (x . w_up[n]) * dm               both projections in one launch
//
// With a handful of tokens the weights' bytes are the whole cost (n*k/2, each used 2m times), so the kernels are
// streams of weights with as little arithmetic per weight as it takes: 8-bit integer products for one or two tokens,
// mma.sync m16n8k16 for a few with few weights, tcgen05 for the rest.  The tensor pipes are far from busy in all of them;
// what the instructions save is issue slots (one weight per lane and FMA would need 8 m of them for 8 weights).  For the
// 16-bit products eight nibbles become four pairs of numbers q - z, exact in either type, with a mask and a multiply-add
// for each.  The sum over a group is an accumulator of 32 bits which is multiplied by the group's scale in fp32: nothing is
// rounded to 16 bits before the result.
//
// Weight blocks.  The fragments fix which lane needs which nibbles, so weights are laid out once for it: 16 rows x 128
// columns are 1 KB in which lane l = 4g + t finds the 32 nibbles of row g (and, 512 bytes on, of row g + 8) that it
// feeds to the block's instructions, as one 16-byte load.  Word u of a lane holds columns 32u + 8t .. +7, so the 4 lanes
// of a row cover 32 columns with each word and a group of 32 never mixes with the next inside one instruction.  The
// scales (and zero points) of those rows and columns follow the codes, and the blocks of 16 rows are contiguous along k:
// a warp reads one stream, whatever the group size.
#include "swiglu_b200.h"

#include <atomic>
#include <type_traits>

#include "launch_common.cuh"
#include "swiglu_kernels.cuh"
#include "tcgen05_common.cuh"

namespace {

using namespace swiglu_b200;

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = kTileRows * kTileCols / 2;
constexpr int kWarps = 8;

// One 4-bit weight matrix in blocks.
struct W4 {
  const void* blocks;  // [row tiles][column tiles]: codes, scales [8][groups][2], zero points likewise in bytes
  int zeros;           // whether blocks have zero points; else they are 8
};

// Bytes of a block.
__host__ __device__ constexpr int block_bytes(int groups, bool zeros) {
  return kTileBytes + groups * 32 + (zeros ? groups * 16 : 0);
}

struct W4Shape {
  long long m, n, k;
  long long x_pitch, y_pitch;  // elements
  int col_tiles;
  int groups_log2;  // log2 of the groups per column tile (0, 1, 2)
  int split;        // CTAs that share a row of column tiles, a cluster
  int row_groups;   // of a cluster (w4_mma_kernel)
  int share, over;  // column tiles (or pairs) of each, and how many of them take one more
  int slice;        // outputs that each finishes
  int y_vec;        // groups of 4 outputs can be stored as one
};

template <class T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
  using V = __nv_bfloat162;
  // A nibble in the low byte of a 16-bit number is that integer times 2^-133 (bf16), wherever it sits in the byte: the
  // subnormals and the first binade go on in equal steps.  One multiply-add brings both places to the same unit and
  // takes the zero point off; all of it is exact.
  static constexpr uint32_t kLow = 0x7f007f00u, kHigh = 0x7d007d00u;  // 2^127, 2^123
  static constexpr float kUnit = 0x1p-6f;
  // Magnitudes above this one, as a float's bits, are whole multiples of 2^(e-156): 8 bits from 2^(e-149) on.
  static __device__ __forceinline__ uint32_t whole_above(int e) { return ((uint32_t)(e - 22) << 23) - 1u; }
  static __device__ __forceinline__ uint32_t pair(float f) {
    __nv_bfloat162 v = __floats2bfloat162_rn(f, f);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float to_float(uint32_t half_word) { return __uint_as_float(half_word << 16); }
  static __device__ __forceinline__ uint16_t from_float(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
  // d = a b + c
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                             float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
};
template <> struct Half2<__half> {
  using V = __half2;
  static constexpr uint32_t kLow = 0x78007800u, kHigh = 0x68006800u;  // 2^15, 2^11; the step of the subnormals is 2^-24
  static constexpr float kUnit = 0x1p-9f;
  // As above with 11 bits; up to e = 132 the unit is no more than 2^-24, of which every number is a multiple.
  static __device__ __forceinline__ uint32_t whole_above(int e) { return e <= 132 ? 0u : ((uint32_t)(e - 19) << 23) - 1u; }
  static __device__ __forceinline__ uint32_t pair(float f) {
    __half2 v = __floats2half2_rn(f, f);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ float to_float(uint32_t half_word) {
    return __half2float(__ushort_as_half((unsigned short)half_word));
  }
  static __device__ __forceinline__ uint16_t from_float(float f) { return __half_as_ushort(__float2half_rn(f)); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                             float c1, float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
};

// Columns (2i, 2i+1) of a word, i = 0..3, as pairs of (q - z) * kUnit; `bias` is the pair -z * kUnit.
template <class T>
__device__ __forceinline__ void weight_pairs(uint32_t word, uint32_t bias, uint32_t (&p)[4]) {
  using H = Half2<T>;
  using V = typename H::V;
  const uint32_t high = word >> 8;
  const uint32_t raw[4] = {word & 0x000f000fu, word & 0x00f000f0u, high & 0x000f000fu, high & 0x00f000f0u};
  const uint32_t low_unit = H::kLow, high_unit = H::kHigh;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    V r = __hfma2(*reinterpret_cast<const V*>(&raw[i]),
                  *reinterpret_cast<const V*>(i & 1 ? &high_unit : &low_unit), *reinterpret_cast<V*>(&bias));
    p[i] = *reinterpret_cast<uint32_t*>(&r);
  }
}

// A zero point 0..15 as a float.
__device__ __forceinline__ float zero_point(uint32_t z) { return __uint_as_float(0x4b000000u | z) - 8388608.0f; }

// Copies from global to shared memory in the calling thread's current group of copies.  copy16 goes past L1 and writes
// zeros behind the first `bytes` bytes, which are all it reads.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes = 16) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() {  // until at most LEFT groups are in flight
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// The `bytes` (a multiple of 16) at `src`, copied by the calling warp; ROUNDS * 512 is at least the largest size.
template <int ROUNDS>
__device__ __forceinline__ void warp_copy(uint32_t dst, const char* src, int bytes, int lane) {
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i)
    if ((i * 32 + lane) * 16 < bytes) copy16(dst + (i * 32 + lane) * 16, src + (i * 32 + lane) * 16);
}

// Launches that follow one another.  A token's projections are launches of a few microseconds in a row, so a launch may
// start while the last CTAs of the one before it (of this file: no other kernel lets it) are still at work.  Until
// `wait_for_previous` it touches no memory but to have its first weights brought to L2; from there on everything that
// was enqueued earlier is complete and visible.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Has `bytes` (a multiple of 16) at `p` brought to L2.
__device__ __forceinline__ void prefetch_l2(const char* p, int bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Clusters.  A launch without one is a cluster of one CTA.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_index() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// The address of `addr` in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_address(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  return remote;
}
// Stores v there and counts its bytes at the barrier at `bar` there.  Waiting for that barrier ends as the last store arrives;
// a cluster barrier that releases the stores takes 0.6 us longer, but many stores go faster uncounted.
__device__ __forceinline__ void cluster_send4(uint32_t addr, uint32_t bar, uint32_t rank, const float4& v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                   cluster_address(addr, rank)),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(cluster_address(bar, rank))
               : "memory");
}
__device__ __forceinline__ void cluster_store4(uint32_t addr, uint32_t rank, const float4& v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_address(addr, rank)), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w)
               : "memory");
}

// Waits for a barrier in the CTA's shared memory; false after half a second.
__device__ __forceinline__ bool own_wait(uint64_t* bar, uint32_t parity) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!tc::mbar_try_wait(bar, parity))
    if (clock64() - t0 > tc::WAIT_CYCLES) return false;
  return true;
}
// A barrier for `bytes` that the cluster sends, made by one thread before the cluster's first barrier.
__device__ __forceinline__ void expect_sums(uint64_t* bar, int bytes) {
  tc::mbar_init(bar, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if (bytes > 0) tc::mbar_expect_tx(bar, bytes);
}

// What a pair of projections (or one alone) comes to.
template <int MATS>
__device__ __forceinline__ float result(const float (&v)[MATS], int activation, const Consts& c) {
  if constexpr (MATS == 1) return v[0];
  else if (activation == ACT_SILU) return Math<true, ACT_SILU>::fwd(v[0], v[1], c);
  else if (activation == ACT_GELU_TANH) return Math<true, ACT_GELU_TANH>::fwd(v[0], v[1], c);
  else return Math<true, ACT_GELU_ERF>::fwd(v[0], v[1], c);
}

// Stores the results of rows n .. n+3, as far as they exist, of the token whose outputs start at `row`.
template <class T, int MATS>
__device__ __forceinline__ void store_results(void* y, long long row, long long n, const W4Shape& s, const float (&v)[4][MATS],
                                              int activation, const Consts& c) {
  uint16_t out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = Half2<T>::from_float(result<MATS>(v[i], activation, c));
  uint16_t* to = static_cast<uint16_t*>(y) + row + n;
  if (s.y_vec && n + 4 <= s.n) {
    *reinterpret_cast<uint2*>(to) = make_uint2(out[0] | (uint32_t)out[1] << 16, out[2] | (uint32_t)out[3] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < s.n) to[i] = out[i];
  }
}

constexpr int kTokenBytes = kTileCols * 2;  // a token's part of a column tile

// ------------------------------------------------------------------ up to 32 tokens, few weights: mma.sync

// Shared memory of a CTA: DEPTH stages of one column tile each, then where the cluster's sums arrive.
template <int MATS, int NT, int GROUPS> struct Cfg {
  static constexpr int SLOT = block_bytes(GROUPS, true);
  static constexpr int WEIGHTS = kWarps * MATS * SLOT, STAGE = WEIGHTS + 8 * NT * kTokenBytes;
  static constexpr int CTAS = 2;  // to an SM
  static constexpr int OUTPUTS = kWarps * kTileRows * 8 * NT;
  static constexpr int ARRIVALS = MATS * (OUTPUTS + 64) * 4;
  static constexpr int FIT = (220 * 1024 / CTAS - ARRIVALS) / STAGE;
  static constexpr int DEPTH = FIT < 3 ? 3 : FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = DEPTH * STAGE + ARRIVALS + 16;  // the last bytes are a barrier
  static_assert(MATS * 8 * NT * (kWarps * kTileRows + 4) * 4 <= DEPTH * STAGE,
                "the sums on their way out reuse the stages");
};

// A CTA owns 8 row tiles (one to a warp; two would read the tokens' fragments once for both, but 128 rows to a CTA
// balance better: fp16 32 x 5504 -> 11009 21.6 us against 23.5) of MATS matrices, up to 8 * NT tokens and, as rank r of a
// cluster of `split` CTAs, the r-th part of the column tiles.  Each rank finishes a slice of the outputs: the others store
// their sums for it into its shared memory, where they are added in a fixed order.
template <class T, int MATS, int NT, int GROUPS>
__global__ void __launch_bounds__(32 * kWarps, Cfg<MATS, NT, GROUPS>::CTAS)
w4_kernel(void* y, const void* __restrict__ x, W4 w0, W4 w1, W4Shape s, int activation, float gm, float dm) {
  using H = Half2<T>;
  using C = Cfg<MATS, NT, GROUPS>;
  constexpr int DEPTH = C::DEPTH, PIECES = 8 * NT * 16, ROUNDS = (PIECES + 32 * kWarps - 1) / (32 * kWarps);
  extern __shared__ __align__(16) unsigned char smem[];
  let_next_start();
  const uint32_t smem_addr = (uint32_t)__cvta_generic_to_shared(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = (int)cluster_rank(), split = s.split;
  const int row_tiles = (int)((s.n + kTileRows - 1) / kTileRows);
  const int row_tile0 = (int)cluster_index() * kWarps, row_tile = row_tile0 + warp;  // of the CTA, the warp
  const int first = rank * s.share + min(rank, s.over), last = first + s.share + (rank < s.over ? 1 : 0);
  const W4 w[2] = {w0, w1};
  // Of the outputs [token][row] that exist each rank finishes `slice` (a multiple of 4).
  constexpr int kRows = kWarps * kTileRows, OUTPUTS = C::OUTPUTS;
  const int outputs = (int)s.m * kRows, slice = s.slice, mine = min(slice, outputs - rank * slice);
  // Whether sums travel as counted stores (us for 4096 -> 4096, uncounted and counted: 5.2 and 4.6 with 8 tokens, 5.7 and 5.6
  // with 12, 7.6 and 7.9 with 32).
  constexpr bool kCounted = NT <= 2;
  // not a variable of its own, which would move all else off its 128-byte boundaries
  uint64_t* const all_arrived = reinterpret_cast<uint64_t*>(smem + C::SMEM - 8);
  if (threadIdx.x == 0) expect_sums(all_arrived, MATS * split * mine * 4);
  cluster_arrive_relaxed();  // all CTAs of the cluster are ready for sums once this is waited for

  const char* src[MATS];  // the warp's next block
#pragma unroll
  for (int a = 0; a < MATS; ++a)
    src[a] = cbyte(w[a].blocks) + ((long long)row_tile * s.col_tiles + first) * block_bytes(GROUPS, w[a].zeros);
  const char* x_src[ROUNDS];  // this thread's pieces of 8 columns of a token, and how many bytes of the row are left there
  long long x_left[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int o = threadIdx.x + i * 32 * kWarps, tok = o >> 4, piece = o & 15;
    const long long k = (long long)first * kTileCols + 8 * piece;
    const bool mine = o < PIECES && tok < s.m;
    x_src[i] = mine ? cbyte(x) + (tok * s.x_pitch + k) * 2 : cbyte(x);
    x_left[i] = mine ? (s.k - k) * 2 : 0;
  }
  int fill = 0;  // offset of the stage to fill next
  // Starts the copies of column tile c; always one group, empty past the last tile.
  auto fetch = [&](int c) {
    if (c < last) {
      const uint32_t stage = smem_addr + fill;
#pragma unroll
      for (int a = 0; a < MATS; ++a) {
        const int bytes = block_bytes(GROUPS, w[a].zeros);
        if (row_tile < row_tiles) warp_copy<(C::SLOT + 511) / 512>(stage + (warp * MATS + a) * C::SLOT, src[a], bytes, lane);
        src[a] += bytes;
      }
      // tokens: every other one has its 64-byte quarters swapped in pairs, so that the 8 lanes that read together (two
      // tokens, four pieces) touch all 32 banks
#pragma unroll
      for (int i = 0; i < ROUNDS; ++i) {
        const int o = threadIdx.x + i * 32 * kWarps, tok = o >> 4, piece = o & 15;
        if (PIECES % (32 * kWarps) == 0 || o < PIECES)
          copy16(stage + C::WEIGHTS + tok * kTokenBytes + (piece ^ ((tok & 1) << 2)) * 16, x_left[i] > 0 ? x_src[i] : cbyte(x),
                 x_left[i] >= 16 ? 16u : x_left[i] > 0 ? (uint32_t)x_left[i] : 0u);
        x_src[i] += kTokenBytes;
        x_left[i] -= kTokenBytes;
      }
    }
    copies_commit();
    fill = fill == (DEPTH - 1) * C::STAGE ? 0 : fill + C::STAGE;
  };

  if (lane < MATS && row_tile < row_tiles) {
    const W4& mine = lane == 0 ? w0 : w1;
    const int bytes = block_bytes(GROUPS, mine.zeros);
    prefetch_l2(cbyte(mine.blocks) + ((long long)row_tile * s.col_tiles + first) * bytes, min(DEPTH - 1, last - first) * bytes);
  }
  wait_for_previous();
#pragma unroll 1
  for (int i = 0; i < DEPTH - 1; ++i) fetch(first + i);

  float acc[MATS][NT][4] = {};
  int take = 0;  // offset of the stage to read next
#pragma unroll 1
  for (int c = first; c < last; ++c) {
    copies_wait<DEPTH - 2>();
    __syncthreads();  // this stage is there for all, and the one before has been read by all
    fetch(c + DEPTH - 1);
    const unsigned char* stage = smem + take;
    take = take == (DEPTH - 1) * C::STAGE ? 0 : take + C::STAGE;
    uint4 codes[MATS][2];
#pragma unroll
    for (int q = 0; q < MATS; ++q)
#pragma unroll
      for (int hi = 0; hi < 2; ++hi)
        codes[q][hi] = *reinterpret_cast<const uint4*>(stage + (warp * MATS + q) * C::SLOT + hi * 512 + lane * 16);
    float part[MATS][NT][4];
    uint32_t bias[MATS][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      constexpr int per_group = 4 / GROUPS;  // words per group
      const int at = (g * GROUPS + u / per_group) * 2;
      uint4 b[NT];  // columns 32u + 8t .. +7 of the tokens, in the pairs that a weight word comes apart into
#pragma unroll
      for (int j = 0; j < NT; ++j)
        b[j] = *reinterpret_cast<const uint4*>(stage + C::WEIGHTS + (8 * j + g) * kTokenBytes +
                                               ((4 * u + t) ^ ((g & 1) << 2)) * 16);
#pragma unroll
      for (int q = 0; q < MATS; ++q) {
        const unsigned char* tail = stage + (warp * MATS + q) * C::SLOT + kTileBytes;
        if (u % per_group == 0) {
          bias[q][0] = bias[q][1] = H::pair(-8.0f * H::kUnit);
          if (w[q].zeros) {
            const uint32_t z = *reinterpret_cast<const uint16_t*>(tail + GROUPS * 32 + at);
            bias[q][0] = H::pair(-H::kUnit * zero_point(z & 0xffu));
            bias[q][1] = H::pair(-H::kUnit * zero_point(z >> 8));
          }
        }
        const uint32_t lo[4] = {codes[q][0].x, codes[q][0].y, codes[q][0].z, codes[q][0].w};
        const uint32_t hi[4] = {codes[q][1].x, codes[q][1].y, codes[q][1].z, codes[q][1].w};
        uint32_t wl[4], wh[4];
        weight_pairs<T>(lo[u], bias[q][0], wl);
        weight_pairs<T>(hi[u], bias[q][1], wh);
        const uint32_t a0[4] = {wl[0], wh[0], wl[1], wh[1]}, a1[4] = {wl[2], wh[2], wl[3], wh[3]};
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float(&p)[4] = part[q][j];
          if (u % per_group == 0) H::mma(p, a0, b[j].x, b[j].y, 0.0f, 0.0f, 0.0f, 0.0f);
          else H::mma(p, a0, b[j].x, b[j].y, p[0], p[1], p[2], p[3]);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float(&p)[4] = part[q][j];
          H::mma(p, a1, b[j].z, b[j].w, p[0], p[1], p[2], p[3]);
        }
        if ((u + 1) % per_group == 0) {
          const uint32_t sc = *reinterpret_cast<const uint32_t*>(tail + at * 2);
          const float scale_lo = H::to_float(sc & 0xffffu), scale_hi = H::to_float(sc >> 16);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[q][j][0] = fmaf(part[q][j][0], scale_lo, acc[q][j][0]);
            acc[q][j][1] = fmaf(part[q][j][1], scale_lo, acc[q][j][1]);
            acc[q][j][2] = fmaf(part[q][j][2], scale_hi, acc[q][j][2]);
            acc[q][j][3] = fmaf(part[q][j][3], scale_hi, acc[q][j][3]);
          }
        }
      }
    }
  }

  copies_wait<0>();
  __syncthreads();  // the stages are done with
  constexpr int kPitch = kRows + 4, kMatrix = 8 * NT * kPitch;  // four tokens of a warp's store hit different banks
  float* sums = reinterpret_cast<float*>(smem);                 // [matrix][token][row]
#pragma unroll
  for (int q = 0; q < MATS; ++q)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)  // row g + 8 (e / 2), token 2t + e % 2 of a tile
        sums[q * kMatrix + (8 * j + 2 * t + e % 2) * kPitch + warp * kTileRows + g + 8 * (e / 2)] =
            acc[q][j][e] * (1.0f / H::kUnit);
  __syncthreads();

  const float* arrived = reinterpret_cast<const float*>(smem + DEPTH * C::STAGE);
  const int begin = split > 1 ? rank * slice : 0;
  bool in_time = true;
  cluster_wait();
  if (split > 1) {
    const uint32_t arrivals = smem_addr + DEPTH * C::STAGE;  // [matrix][rank][slice]
#pragma unroll 1
    for (int o = 4 * threadIdx.x; o < outputs; o += 128 * kWarps) {
      const int owner = (int)((unsigned)o / (unsigned)slice), at = rank * slice + o - owner * slice;
#pragma unroll
      for (int a = 0; a < MATS; ++a) {
        const uint32_t to = arrivals + (a * (OUTPUTS + 64) + at) * 4;
        const float4& v = *reinterpret_cast<const float4*>(sums + a * kMatrix + o / kRows * kPitch + o % kRows);
        if constexpr (kCounted) cluster_send4(to, tc::smem_u32(all_arrived), owner, v);
        else cluster_store4(to, owner, v);
      }
    }
    if constexpr (kCounted) {
      in_time = mine <= 0 || own_wait(all_arrived, 0);
    } else {
      cluster_arrive();
      cluster_wait();
    }
  }
  const Consts consts(gm, dm);
#pragma unroll 1
  for (int o = 4 * threadIdx.x; o < mine; o += 128 * kWarps) {
    const int row = (begin + o) % kRows, tok = (begin + o) / kRows;
    const long long n = (long long)row_tile0 * kTileRows + row;
    if (n >= s.n) continue;
    float v[4][MATS];
#pragma unroll
    for (int a = 0; a < MATS; ++a) {
      const float* p = split > 1 ? arrived + a * (OUTPUTS + 64) + o : sums + a * kMatrix + tok * kPitch + row;
      float4 f = *reinterpret_cast<const float4*>(p);
#pragma unroll 1
      for (int i = 1; i < split; ++i) {
        const float4 add = *reinterpret_cast<const float4*>(p + i * slice);
        f.x += add.x, f.y += add.y, f.z += add.z, f.w += add.w;
      }
      v[0][a] = f.x, v[1][a] = f.y, v[2][a] = f.z, v[3][a] = f.w;
    }
    if (!in_time) v[0][0] = v[1][0] = v[2][0] = v[3][0] = __uint_as_float(0x7fffffffu);
    store_results<T, MATS>(y, tok * s.y_pitch, n, s, v, activation, consts);
  }
}

// ------------------------------------------------------------------ more tokens or weights: tcgen05
//
// 128 rows of weights are the M of tcgen05.mma, 16, 32 or 64 tokens its N.  A thread keeps one row: it reads the 64 bytes
// of codes that the row has in a block, turns them into pairs of 16-bit numbers as above and stores them as A in its lane
// of the tensor memory, from where the tensor core reads them; the tokens are B, which it reads from shared memory as a
// tiled copy has laid them out.  Against mma.sync no warp reads tokens any more (with 32 of them that was 64 of the 82
// accesses to shared memory for a block), and the work for a weight is the same for any number of tokens.  The products
// of a scale group are read back, and scaled and added up in registers.
//
// A CTA takes an SM to itself (all 512 columns of tensor memory, 224 KB of stages) and has four such warpgroups, which work on
// column tiles of their own.  While one waits for its products the others turn codes into numbers; what bounds the kernel
// are the instructions for that (bf16 32 x 4096 -> 14336 gate and up: 84 % of the issue slots of the busy SMs).

constexpr int kGroupThreads = 128, kGroups = 4;  // warpgroups, a thread to a weight row
constexpr int kGroupRows = 128;

// Distance of the blocks of a column tile in shared memory: an odd multiple of 16, so that four of them start in different
// banks.  The copies bring what follows a block along.
__host__ __device__ constexpr int slot_bytes(int groups, bool zeros) { return block_bytes(groups, zeros) | 16; }

// What w4_mma_kernel copies from: the tokens, and each matrix as [row tiles][bytes] in elements of 8 bytes.
struct Maps {
  CUtensorMap x, w[2];
};

// Shared memory of a CTA: DEPTH stages of each warpgroup's column tile of the tokens, then of its blocks; where the
// cluster's sums arrive takes the place of the stages.
template <int N, int GROUPS> struct MmaCfg {
  static constexpr int SLOT = slot_bytes(GROUPS, true);
  static constexpr int X = N * kTokenBytes, TILES = kGroupRows / kTileRows;
  // swizzled tiles start on multiples of 1024
  static constexpr int STAGE = (kGroups * (X + TILES * SLOT) + 1023) / 1024 * 1024;
  static constexpr int FIT = 224 * 1024 / STAGE, DEPTH = FIT > 6 ? 6 : FIT;
  static constexpr int SMEM = 1024 + DEPTH * STAGE;  // the first kilobyte is lost to alignment
  static constexpr int A_COLS = kTileCols / 2, D_COLS = 64, TMEM = kGroups * (A_COLS + D_COLS);
  static constexpr int AT_ONCE = D_COLS / N < GROUPS ? D_COLS / N : GROUPS;  // groups whose products are held at a time
  // the cluster's sums take the place of the stages: those that arrive, and as many tokens of those that leave as fit
  static constexpr int ARRIVALS = (kGroups * N + 32) * kGroupRows * 4, LEAVING = N < 64 ? N : 16;
  static_assert(DEPTH >= 2 && ARRIVALS + kGroups * LEAVING * kGroupRows * 4 <= DEPTH * STAGE, "room for the sums");
};

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// D (+)= A B with A in tensor memory
__device__ __forceinline__ void mma_from_tmem(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a),
      "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tile_load(uint32_t dst, const CUtensorMap& map, int col, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(&map), "r"(col), "r"(row), "r"(tc::smem_u32(bar))
      : "memory");
}
// True for one lane of a warp whose lanes all take part.
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void group_sync(int group) {  // of a warpgroup
  asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(kGroupThreads) : "memory");
}

// A cluster of `split` CTAs owns `row_groups` times 128 rows of MATS matrices and N tokens.
template <class T, int MATS, int N, int GROUPS>
__global__ void __launch_bounds__(kGroups * kGroupThreads, 1)
w4_mma_kernel(void* y, const __grid_constant__ Maps maps, W4 w0, W4 w1, W4Shape s, int activation, float gm, float dm) {
  using H = Half2<T>;
  using C = MmaCfg<N, GROUPS>;
  constexpr int DEPTH = C::DEPTH, TILES = C::TILES;
  extern __shared__ unsigned char raw_smem[];
  __shared__ uint32_t tmem_slot;
  __shared__ __align__(8) uint64_t products[kGroups], full[kGroups][DEPTH];
  let_next_start();
  const uint32_t smem_addr = ((uint32_t)__cvta_generic_to_shared(raw_smem) + 1023u) & ~1023u;
  unsigned char* smem = raw_smem + (smem_addr - (uint32_t)__cvta_generic_to_shared(raw_smem));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, quarter = warp & 3;
  const int group = warp >> 2;  // the warpgroup
  // A thread's lane of the tensor memory, and the row of the weights that it holds.  Any order of the rows will do; in
  // this one the eight threads that read together touch two rows of each of four blocks, which are in different banks.
  const int tile = (quarter >> 1) * 4 + (lane & 3), in_tile = (quarter & 1) * 8 + (lane >> 2), row = tile * kTileRows + in_tile;
  // The cluster's row groups and matrices are dealt to its warpgroups, `parts` of them to each, which share its column tiles.
  const int rank = (int)cluster_rank(), worker = rank * kGroups + group, jobs = s.row_groups * MATS;
  const int part = worker / jobs, parts = s.split * kGroups / jobs, job = worker - part * jobs;
  const int matrix = job % MATS, row_group = job / MATS;  // the latter in the cluster
  const int row_tiles = (int)((s.n + kTileRows - 1) / kTileRows);
  const int row_tile0 = ((int)cluster_index() * s.row_groups + row_group) * TILES;
  const int tiles = max(0, min(TILES, row_tiles - row_tile0));
  const int token0 = (int)blockIdx.y * N;
  const W4 w = matrix ? w1 : w0;
  const int bytes = block_bytes(GROUPS, w.zeros);
  const int share = s.col_tiles / parts, over = s.col_tiles % parts;
  const int first = part * share + min(part, over), last = tiles > 0 ? first + share + (part < over ? 1 : 0) : first;
  const int tokens = s.m - token0 < N ? (int)(s.m - token0) : N;

  const uint32_t w_at = kGroups * C::X + group * TILES * C::SLOT;  // in a stage
  const int slot = slot_bytes(GROUPS, w.zeros);
  int fill = 0;  // the stage to fill next
  // Starts the copies of column tile c, from one thread of the warpgroup's second warp: an instruction takes about a hundred
  // cycles to leave, and this warp has nothing to do while the first one starts the products.
  auto fetch = [&](int c) {
    if (elect()) {
      uint64_t* bar = &full[group][fill];
      const uint32_t to = smem_addr + fill * C::STAGE;
      tc::mbar_expect_tx(bar, C::X + TILES * slot);
      tile_load(to + w_at, maps.w[matrix], c * (bytes / 8), row_tile0, bar);
      tile_load(to + group * C::X, maps.x, c * kTileCols, token0, bar);
      tile_load(to + group * C::X + N * 128, maps.x, c * kTileCols + 64, token0, bar);
    }
    fill = fill == DEPTH - 1 ? 0 : fill + 1;
  };

  if (threadIdx.x % kGroupThreads < tiles && first < last)
    prefetch_l2(cbyte(w.blocks) + ((long long)(row_tile0 + (int)threadIdx.x % kGroupThreads) * s.col_tiles + first) * bytes,
                min(DEPTH, last - first) * bytes);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kGroups; ++i) {
      tc::mbar_init(&products[i], 1);
      for (int d = 0; d < DEPTH; ++d) tc::mbar_init(&full[i][d], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  wait_for_previous();
  if (quarter == 1 && first < last) fetch(first);
  __syncwarp();
  // Only now: a launch that waits for the one before it must not hold tensor memory which that one still asks for.  It
  // is given back before the CTA waits for any other.
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&tmem_slot)),
                 "n"(C::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0) + group * (C::A_COLS + C::D_COLS);
  const uint32_t tmem_row = tmem + ((uint32_t)(quarter * 32) << 16);
  constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t idesc = (1u << 4) | (type << 7) | (type << 10) | ((N >> 3) << 17) | ((128u >> 4) << 24);

  if (quarter == 1) {
#pragma unroll 1
    for (int i = 1; i < DEPTH && first + i < last; ++i) fetch(first + i);
  }
  float acc[N] = {};
  bool ok = true;
  uint32_t parity = 0;
  int take = 0, round = 0;  // the stage to read next, and how often it has been filled before, modulo 2
#pragma unroll 1
  for (int c = first; c < last; ++c) {
    ok = ok && own_wait(&full[group][take], round);
    const unsigned char* block = smem + w_at + take * C::STAGE + tile * slot;
    const unsigned char* tail = block + kTileBytes;
    const int at = (in_tile & 7) * GROUPS * 2 + (in_tile >> 3);  // of the first group's scale
    uint4 codes[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) codes[t] = *reinterpret_cast<const uint4*>(block + in_tile * 64 + t * 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      constexpr int per_group = 4 / GROUPS;  // words per group
      uint32_t bias = H::pair(-8.0f * H::kUnit);
      if (w.zeros) bias = H::pair(-H::kUnit * zero_point(tail[GROUPS * 32 + at + u / per_group * 2]));
      uint32_t a[16];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t words[4] = {codes[t].x, codes[t].y, codes[t].z, codes[t].w};
        uint32_t p[4];
        weight_pairs<T>(words[u], bias, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[4 * t + i] = p[i];
      }
      tmem_st16(tmem_row + 16 * u, a);
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
#pragma unroll
    for (int g0 = 0; g0 < GROUPS; g0 += C::AT_ONCE) {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      group_sync(group);  // all of A and of the tokens is there, what D held has been read
      if (quarter == 0) {
        if (elect()) {
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint64_t b = tc::umma_desc(smem_addr + group * C::X + take * C::STAGE);
#pragma unroll
          for (int g = 0; g < C::AT_ONCE; ++g)
#pragma unroll
            for (int i = 0; i < 8 / GROUPS; ++i) {  // 16 columns each
              const int kk = (g0 + g) * (8 / GROUPS) + i;
              mma_from_tmem(tmem + C::A_COLS + g * N, tmem + 8 * kk, b + (kk >> 2) * (N * 128 / 16) + 2 * (kk & 3), idesc,
                            i != 0);
            }
          tc::umma_commit(&products[group]);
        }
      } else if (quarter == 1 && g0 == 0 && c > first && c - 1 + DEPTH < last) {
        fetch(c - 1 + DEPTH);  // the stage before this one has been read by all
      }
      __syncwarp();
      ok = ok && own_wait(&products[group], parity);
      parity ^= 1;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
      for (int g = 0; g < C::AT_ONCE; ++g) {
        const float scale = H::to_float(*reinterpret_cast<const uint16_t*>(tail + (at + (g0 + g) * 2) * 2));
        constexpr int STEP = N < 32 ? 16 : 32;
#pragma unroll
        for (int j0 = 0; j0 < N; j0 += STEP) {
          uint32_t d[STEP];
          if constexpr (STEP == 16) tc::tmem_ld16(tmem_row + C::A_COLS + g * N + j0, d);
          else tc::tmem_ld32(tmem_row + C::A_COLS + g * N + j0, d);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int j = 0; j < STEP; ++j) acc[j0 + j] = fmaf(__uint_as_float(d[j]), scale, acc[j0 + j]);
        }
      }
    }
    if (++take == DEPTH) {
      take = 0;
      round ^= 1;
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  const bool failed = __syncthreads_or(!ok);
  if (failed) {  // copies and products may still be under way
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {
    }
  }
  cluster_arrive_relaxed();  // nothing was written for the others yet
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "n"(C::TMEM) : "memory");
  }
  cluster_wait();  // no CTA of the cluster needs its stages any more
  // Each rank finishes `slice` of the cluster's [row group][token].  What arrives there: [matrix][part][of the slice][row].
  const int slice = s.slice;
  const int mine = min(slice, s.row_groups * tokens - rank * slice);
  const float unit = failed ? __uint_as_float(0x7fffffffu) : 1.0f / H::kUnit;
  const uint32_t to = smem_addr + (matrix * parts + part) * slice * (kGroupRows * 4) + lane * 16;
  unsigned char* leaving = smem + C::ARRIVALS + group * (C::LEAVING * kGroupRows * 4);  // [token][row] of this warpgroup
#pragma unroll
  for (int j0 = 0; j0 < N; j0 += C::LEAVING) {
    if (j0 != 0) group_sync(group);
#pragma unroll
    for (int j = 0; j < C::LEAVING; ++j) *reinterpret_cast<float*>(leaving + (j * kGroupRows + row) * 4) = acc[j0 + j] * unit;
    group_sync(group);
#pragma unroll 1
    for (int j = quarter; j < C::LEAVING && j0 + j < tokens; j += 4) {  // a warp to a token
      const int i = row_group * tokens + j0 + j, owner = i / slice;
      cluster_store4(to + (i - owner * slice) * (kGroupRows * 4), owner,
                     *reinterpret_cast<const float4*>(leaving + j * (kGroupRows * 4) + lane * 16));
    }
  }
  cluster_arrive();
  cluster_wait();
  const Consts consts(gm, dm);
#pragma unroll 1
  for (int o = warp; o < mine; o += kGroups * 4) {  // a warp to a token, a lane to four rows
    const int unit_row = (rank * slice + o) / tokens, token = (rank * slice + o) - unit_row * tokens;
    const long long n = ((long long)cluster_index() * s.row_groups + unit_row) * kGroupRows + 4 * lane;
    if (n >= s.n) continue;
    float v[4][MATS] = {};
#pragma unroll 1
    for (int i = 0; i < parts; ++i)
#pragma unroll
      for (int a = 0; a < MATS; ++a) {
        const float4 f =
            *reinterpret_cast<const float4*>(smem + ((a * parts + i) * slice + o) * (kGroupRows * 4) + lane * 16);
        v[0][a] += f.x, v[1][a] += f.y, v[2][a] += f.z, v[3][a] += f.w;
      }
    store_results<T, MATS>(y, ((long long)token0 + token) * s.y_pitch, n, s, v, activation, consts);
  }
}

// ------------------------------------------------------------------ one or two tokens: digits and integer products

// As bytes the 8 nibbles of a word are two registers after three instructions (9 and four multiply-adds above), and
// m16n8k32 multiplies them as they are.  For that a token is written as four 8-bit digits of a 31-bit number: with 2^e
// above the largest magnitude of its 256 columns (a span), X = x * 2^(30-e) = d0 + 2^8 d1 + 2^16 d2 + 2^24 d3, the digits
// balanced around zero.  Its digits are four columns of the product, so two tokens fill the eight columns of one
// instruction.  Within a group the sums of nibble * digit are exact in 32 bits, the zero point comes off as z times the
// digits' own sum (exact as well), and what is left, below 2^19, goes on in fp32: times the group's scale and 2^(8i+e-30).
//
// X is a whole number, nothing of x is lost, for bf16 within 2^22 of the largest magnitude of the span and for fp16 within
// 2^19, or wherever that magnitude is below 64.  It has to be: where the weight of a large column is zero, the small ones
// beside it are the result.  A single token has the other four columns as well, for the digits of what X leaves over,
// another 31 bits below.  With two tokens, or where 62 bits are too few (or the numbers below 2^-63, whose unit would leave
// fp32, or not finite), the span takes the 16-bit products of the kernels above, with the weights where they are: its unit is zero as a
// mark, so its digits add nothing.
//
// us without such a span / with one / with one in every span: bf16 1 x 14336 -> 4096 7.9 / 8.2 / 8.7, gate and up
// 1 x 4096 -> 14336 13.0 / 13.2 / 13.8, two tokens 4096 -> 11008 13.3 / 16.5 / 31.2.  Products silu(g) u of normal numbers
// have one in 0.3 % of their spans in bf16 and in none in fp16.

constexpr int kDigitTokens = 2, kDigits = 4, kDigitCols = kDigits * kDigitTokens;
constexpr int kSlab = 16;                              // column tiles whose digits are kept at a time, in pairs

// A CTA: ROW_WARPS row tiles, whose pairs of column tiles are dealt to the warps that are left over.
template <int MATS, int GROUPS, int ROW_WARPS> struct DigitCfg {
  static constexpr int COL_WARPS = kWarps / ROW_WARPS, OUTPUTS = ROW_WARPS * kTileRows * kDigitTokens;
  // A pair of blocks, as far from a 128-byte boundary as it is in the weights: copies between unlike places cost more (half
  // a sector apart 1 x 4096 -> 14336 takes 16.9 us, whole sectors 13.9, this 13.5).
  static constexpr int SLOT = (2 * block_bytes(GROUPS, true) + 127) / 128 * 128 + 128;
  static constexpr int PAIR = MATS * SLOT;
  static constexpr int DEPTH = MATS == 1 ? 4 : 2;                 // pairs of a warp in flight
  static constexpr int RING = kWarps * DEPTH * PAIR;
  static constexpr int DIGITS = kSlab * 2 * kDigitCols * 4 * 16;  // [tile][2][column][t] 16 bytes
  static constexpr int SUMS = kSlab * GROUPS * 8 * 4;             // [tile][group][8]
  static constexpr int UNITS = kSlab / 2 * 8 * 4;                 // [pair][8]
  static constexpr int ARRIVALS = MATS * COL_WARPS * (OUTPUTS + 64) * 4;  // [matrix][column warp][rank][slice]
  static constexpr int SMEM = RING + DIGITS + SUMS + UNITS + ARRIVALS + 16;  // the last bytes are a barrier
};

__device__ __forceinline__ void imma(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr float kIntMagic = 12582912.0f;  // 1.5 * 2^23: added to an integer below 2^22, its bits are 0x4b400000 + it
constexpr uint32_t kIntMagicBits = 0x4b400000u;

// The 16-bit products of a span.  `block` is its first block of weights in shared memory, one of `tiles`; at `token` is the
// place of its digits, where those of a marked token are the token itself, 16 bytes where the first two digits of its
// eight columns would be.  Column g of B is token g; those whose bit 2 g is not in `marked` are zero.  The sums, of rows g and
// g + 8 in units of kUnit, are returned to the lanes that hold the first digits: to t = 0 token 0's, to t = 2 token 1's.
// A function of its own: as a part of the loop that rarely calls it, it took that 5 % of its time.
template <class T, int GROUPS>
__device__ __noinline__ float2 span_products(const unsigned char* block, bool zeros, const unsigned char* token, int tiles,
                                             uint32_t marked) {
  using H = Half2<T>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool mine = g < kDigitTokens && marked >> (2 * g) & 1;
  token += ((g & 1) * kDigits * 4 + t) * 16;
  float sum[4] = {};
#pragma unroll 1
  for (int h = 0; h < tiles; ++h, block += block_bytes(GROUPS, zeros), token += 2 * kDigitCols * 64)
#pragma unroll
  for (int u = 0; u < 4; ++u) {  // 32 columns each
    const int at = (g * GROUPS + u * GROUPS / 4) * 2;
    const unsigned char* tail = block + kTileBytes;
    const uint4 b = mine ? *reinterpret_cast<const uint4*>(token + ((u >> 1) * kDigitCols + (u & 1)) * 64)
                         : make_uint4(0u, 0u, 0u, 0u);
    uint32_t bias_lo = H::pair(-8.0f * H::kUnit), bias_hi = bias_lo;
    if (zeros) {
      const uint32_t z = *reinterpret_cast<const uint16_t*>(tail + GROUPS * 32 + at);
      bias_lo = H::pair(-H::kUnit * zero_point(z & 0xffu));
      bias_hi = H::pair(-H::kUnit * zero_point(z >> 8));
    }
    uint32_t wl[4], wh[4];
    weight_pairs<T>(*reinterpret_cast<const uint32_t*>(block + lane * 16 + 4 * u), bias_lo, wl);
    weight_pairs<T>(*reinterpret_cast<const uint32_t*>(block + 512 + lane * 16 + 4 * u), bias_hi, wh);
    const uint32_t a0[4] = {wl[0], wh[0], wl[1], wh[1]}, a1[4] = {wl[2], wh[2], wl[3], wh[3]};
    float part[4];
    H::mma(part, a0, b.x, b.y, 0.0f, 0.0f, 0.0f, 0.0f);
    H::mma(part, a1, b.z, b.w, part[0], part[1], part[2], part[3]);
    const uint32_t sc = *reinterpret_cast<const uint32_t*>(tail + at * 2);
    const float s_lo = H::to_float(sc & 0xffffu), s_hi = H::to_float(sc >> 16);
    sum[0] = fmaf(part[0], s_lo, sum[0]);
    sum[1] = fmaf(part[1], s_lo, sum[1]);
    sum[2] = fmaf(part[2], s_hi, sum[2]);
    sum[3] = fmaf(part[3], s_hi, sum[3]);
  }
  // the lanes t = 0 have the sums of both tokens
  const float lo = __shfl_sync(0xffffffffu, sum[1], lane & 28), hi = __shfl_sync(0xffffffffu, sum[3], lane & 28);
  return t == 0 ? make_float2(sum[0], sum[2]) : t == 2 ? make_float2(lo, hi) : make_float2(0.0f, 0.0f);
}

// A CTA owns ROW_WARPS row tiles of MATS matrices, up to two tokens and, as rank r of a cluster of `split` CTAs, the
// r-th part of the pairs of column tiles.  The code is kept short (loops that are not unrolled): a launch lasts a few
// microseconds, most of its instructions run once, and a start waits for them to be fetched.
template <class T, int MATS, int GROUPS, int ROW_WARPS>
__global__ void __launch_bounds__(32 * kWarps, 2)
w4_digits_kernel(void* y, const void* __restrict__ x, W4 w0, W4 w1, W4Shape s, int activation, float gm, float dm) {
  using H = Half2<T>;
  using C = DigitCfg<MATS, GROUPS, ROW_WARPS>;
  constexpr int DEPTH = C::DEPTH, COL_WARPS = C::COL_WARPS;
  extern __shared__ __align__(16) unsigned char smem[];
  let_next_start();
  // not a variable of its own, which would move all else off its 128-byte boundaries
  uint64_t* const sums = reinterpret_cast<uint64_t*>(smem + C::SMEM - 8);
  const uint32_t smem_addr = (uint32_t)__cvta_generic_to_shared(smem);
  unsigned char* digits = smem + C::RING;
  float* digit_sums = reinterpret_cast<float*>(digits + C::DIGITS);
  float* units = reinterpret_cast<float*>(digits + C::DIGITS + C::SUMS);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row_warp = warp % ROW_WARPS, col_warp = warp / ROW_WARPS;
  const int rank = (int)cluster_rank(), split = s.split;
  const int first = rank * s.share + min(rank, s.over), last = first + s.share + (rank < s.over ? 1 : 0);  // pairs
  const int row_tile0 = (int)cluster_index() * ROW_WARPS, row_tile = row_tile0 + row_warp;  // of the CTA, the warp
  const bool there = (long long)row_tile * kTileRows < s.n;
  const int tokens = (int)s.m;
  const W4 w[2] = {w0, w1};
  constexpr int kRows = ROW_WARPS * kTileRows;
  // Each rank finishes `slice` (a multiple of 4) of the outputs [token][row].
  const int outputs = tokens * kRows, slice = s.slice;
  const int mine = min(slice, outputs - rank * slice);
  if (threadIdx.x == 0) expect_sums(sums, MATS * COL_WARPS * split * mine * 4);
  cluster_arrive_relaxed();  // all CTAs of the cluster are ready for sums once this is waited for

  // This thread's eight columns of a token, of the slab that starts at pair p; zeros past the last one.
  auto read_token = [&](int p, int tok) {
    const long long k = (long long)p * (2 * kTileCols) + 8 * threadIdx.x;
    const char* src = cbyte(x) + (tok * s.x_pitch + k) * 2;
    Vec<16> v{};
    if (k + 8 <= s.k) {
      v = Ld<16, LD_PLAIN>::ld(src);
    } else {
#pragma unroll 1
      for (int e = 0; k + e < s.k; ++e) {
        const uint32_t bits = Ld<2, LD_PLAIN>::ld(src + 2 * e).w[0] << (16 * (e & 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[i] |= e / 2 == i ? bits : 0u;
      }
    }
    return v;
  };
  // Writes the digits of part `part` of a span, `f`: with two tokens a part is a token, with one it is the token and then what
  // its digits left over.  A warp holds one span.  True when there is another part, which is then in `f` with one token.
  auto write_digits = [&](const Vec<16>& token, float (&f)[8], int part) {
    const int piece = threadIdx.x & 15, tile = threadIdx.x >> 4, u = piece >> 2;
    uint32_t top = 0, below = 0xffffffffu;  // the largest magnitude, the least one but zero less one
#pragma unroll
    for (int a = 0; a < 8; ++a) {
      const uint32_t magnitude = __float_as_uint(f[a]) & 0x7fffffffu;
      top = max(top, magnitude);
      below = min(below, magnitude - 1u);
    }
    const int e = max((int)(__reduce_max_sync(0xffffffffu, top) >> 23), 64);  // the magnitudes are below 2^(e - 126)
    const float up = __uint_as_float((uint32_t)(283 - e) << 23);  // 2^(156-e)
    const bool whole = __all_sync(0xffffffffu, below >= H::whole_above(e)) && e != 255;
    uint32_t z[8];  // bytes: the digits
#pragma unroll
    for (int a = 0; a < 8; ++a) z[a] = ((uint32_t)__float2int_rn(f[a] * up) + 0x80808080u) ^ 0x80808080u;
    const bool marked = !whole && (part + 1 >= kDigitTokens / tokens || e == 255);
    if (const int d = lane - kDigits * part; lane < kDigitCols && (d >= 0 || (marked && tokens == 1)))
      units[warp * kDigitCols + lane] = marked || d >= kDigits ? 0.0f : __uint_as_float((uint32_t)(e - 29 + 8 * d) << 23);
    // digits of four columns to a word, in the order of the nibbles: even ones columns 0, 4, 1, 5, odd ones 2, 6, 3, 7
    uint32_t digit[2][kDigits];
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const uint32_t a0 = __byte_perm(z[2 * odd], z[2 * odd + 4], 0x5140), a1 = __byte_perm(z[2 * odd], z[2 * odd + 4], 0x7362);
      const uint32_t b0 = __byte_perm(z[2 * odd + 1], z[2 * odd + 5], 0x5140);
      const uint32_t b1 = __byte_perm(z[2 * odd + 1], z[2 * odd + 5], 0x7362);
      digit[odd][0] = __byte_perm(a0, b0, 0x5410);
      digit[odd][1] = __byte_perm(a0, b0, 0x7632);
      digit[odd][2] = __byte_perm(a1, b1, 0x5410);
      digit[odd][3] = __byte_perm(a1, b1, 0x7632);
    }
    unsigned char* to = digits + ((tile * 2 + (u >> 1)) * kDigitCols * 4 + (piece & 3)) * 16;
    int total[kDigits];
#pragma unroll
    for (int d = 0; d < kDigits; ++d) {
      total[d] = __dp4a((int)digit[0][d], 0x01010101, __dp4a((int)digit[1][d], 0x01010101, 0));
      if (!marked)
        *reinterpret_cast<uint2*>(to + (kDigits * part + d) * 64 + (u & 1) * 8) = make_uint2(digit[0][d], digit[1][d]);
    }
    if (marked) {
      __syncwarp();  // over the first part's digits, other lanes' among them
      *reinterpret_cast<uint4*>(to + ((tokens == 1 ? 0 : kDigits * part) + (u & 1)) * 64) =
          make_uint4(token.w[0], token.w[1], token.w[2], token.w[3]);
    }
    // sums over the 4, 8 or 16 threads of a group; two of them travel in one register (each below 2^15)
    int low = total[0] + (total[1] << 16), high = total[2] + (total[3] << 16);
#pragma unroll
    for (int d = 1; d < 16 / GROUPS; d *= 2) {
      low += __shfl_xor_sync(0xffffffffu, low, d);
      high += __shfl_xor_sync(0xffffffffu, high, d);
    }
    if (piece % (16 / GROUPS) == 0)
      *reinterpret_cast<float4*>(digit_sums + (threadIdx.x / (16 / GROUPS)) * kDigitCols + kDigits * part) =
          make_float4((float)(short)low, (float)((low - (short)low) >> 16), (float)(short)high,
                      (float)((high - (short)high) >> 16));
    if (part == 1 || tokens == 2) return part == 0;
    if (whole || marked) return false;
    const float down = __uint_as_float((uint32_t)(e - 29) << 23);
#pragma unroll
    for (int a = 0; a < 8; ++a) f[a] = fmaf(-(float)__float2int_rn(f[a] * up), down, f[a]);  // a difference of multiples of its last bit
    return true;
  };

  // The warp's ring of pairs of blocks.
  const unsigned char* ring = smem + warp * (DEPTH * C::PAIR);
  const uint32_t ring_addr = smem_addr + warp * (DEPTH * C::PAIR);
  const char* src[MATS];  // the warp's next pair
  uint32_t place[MATS];   // where the pair to read next was, modulo 2^32
#pragma unroll
  for (int a = 0; a < MATS; ++a) {
    src[a] = cbyte(w[a].blocks) +
             ((long long)row_tile * s.col_tiles + 2 * (first + col_warp)) * block_bytes(GROUPS, w[a].zeros);
    place[a] = (uint32_t)(uintptr_t)src[a];
  }
  int fill = 0;  // offset of the slot to fill next
  auto fetch = [&](int p) {  // always one group of copies, empty past the last pair
    if (p < last && there) {
#pragma unroll
      for (int a = 0; a < MATS; ++a) {
        const int bytes = block_bytes(GROUPS, w[a].zeros);
        warp_copy<(2 * block_bytes(GROUPS, true) + 511) / 512>(
            ring_addr + fill + a * C::SLOT + ((uint32_t)(uintptr_t)src[a] & 127u), src[a],
            2 * p + 1 == s.col_tiles ? bytes : 2 * bytes, lane);
        src[a] += 2 * COL_WARPS * bytes;
      }
    }
    copies_commit();
    fill = fill == (DEPTH - 1) * C::PAIR ? 0 : fill + C::PAIR;
  };

  if (lane < MATS && there && first < last) {
    const W4& mine = lane == 0 ? w0 : w1;
    const int bytes = block_bytes(GROUPS, mine.zeros);
    // the column warps of a row ask for the same few pairs
    prefetch_l2(cbyte(mine.blocks) + ((long long)row_tile * s.col_tiles + 2 * first) * bytes,
                min((DEPTH - 1) * COL_WARPS * 2, min(2 * last, s.col_tiles) - 2 * first) * bytes);
  }
  // sums of the second part's digits where there is none: its unit is zero, and these have to be finite
  if (tokens == 1 && threadIdx.x % (16 / GROUPS) == 0)
    *reinterpret_cast<float4*>(digit_sums + (threadIdx.x / (16 / GROUPS)) * kDigitCols + kDigits) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  wait_for_previous();
  Vec<16> token = read_token(first, 0);
#pragma unroll 1
  for (int i = 0; i < DEPTH - 1; ++i) fetch(first + col_warp + i * COL_WARPS);

  float acc[MATS][4] = {};
  int take = 0;  // offset of the slot to read next
#pragma unroll 1
  for (int slab = first; slab < last; slab += kSlab / 2) {
    if (slab != first) {
      __syncthreads();  // the digits have been read by all
      token = read_token(slab, 0);
    }
    float f[8];
    Codec<T>::template unpack<16>(token, f);
#pragma unroll 1
    for (int part = 0; write_digits(token, f, part); ++part)
      if (tokens == 2) {
        token = read_token(slab, 1);
        Codec<T>::template unpack<16>(token, f);
      }
    __syncthreads();
    const int end = last < slab + kSlab / 2 ? last : slab + kSlab / 2;
#pragma unroll 1
    for (int p = slab + col_warp; p < end; p += COL_WARPS) {
      copies_wait<DEPTH - 2>();
      __syncwarp();  // this pair is there for all lanes, and the one before has been read by all
      fetch(p + (DEPTH - 1) * COL_WARPS);
      if (!there) continue;
      const float2 unit = *reinterpret_cast<const float2*>(units + (p - slab) * 8 + 2 * t);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (2 * p + h == s.col_tiles) break;
        const int in_slab = 2 * (p - slab) + h;
        const unsigned char* piece = digits + (in_slab * 2 * kDigitCols * 4 + lane) * 16;
        const uint4 b0 = *reinterpret_cast<const uint4*>(piece);
        const uint4 b1 = *reinterpret_cast<const uint4*>(piece + kDigitCols * 64);
        const uint32_t b[4][2] = {{b0.x, b0.y}, {b0.z, b0.w}, {b1.x, b1.y}, {b1.z, b1.w}};
#pragma unroll
        for (int a = 0; a < MATS; ++a) {
          const unsigned char* slot = ring + take + a * C::SLOT + (place[a] & 127u) + h * block_bytes(GROUPS, w[a].zeros);
          const uint4 lo4 = *reinterpret_cast<const uint4*>(slot + lane * 16);
          const uint4 hi4 = *reinterpret_cast<const uint4*>(slot + 512 + lane * 16);
          const uint32_t lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
          uint32_t d[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            constexpr int per_group = 4 / GROUPS;  // words per group
            if (u % per_group == 0) d[0] = d[1] = d[2] = d[3] = kIntMagicBits;
            imma(d, lo[u] & 0x0f0f0f0fu, hi[u] & 0x0f0f0f0fu, lo[u] >> 4 & 0x0f0f0f0fu, hi[u] >> 4 & 0x0f0f0f0fu,
                 b[u][0], b[u][1]);
            if ((u + 1) % per_group == 0) {
              const int at = (g * GROUPS + u / per_group) * 2;
              const uint32_t sc = *reinterpret_cast<const uint32_t*>(slot + kTileBytes + at * 2);
              const float s_lo = H::to_float(sc & 0xffffu), s_hi = H::to_float(sc >> 16);
              float z_lo = 8.0f, z_hi = 8.0f;
              if (w[a].zeros) {
                const uint32_t z = *reinterpret_cast<const uint16_t*>(slot + kTileBytes + GROUPS * 32 + at);
                z_lo = zero_point(z & 0xffu);
                z_hi = zero_point(z >> 8);
              }
              const float2 sum = *reinterpret_cast<const float2*>(digit_sums + (in_slab * GROUPS + u / per_group) * 8 + 2 * t);
              // every term in front of the scale is an integer below 2^24: exact
              acc[a][0] = fmaf(__uint_as_float(d[0]) + fmaf(-z_lo, sum.x, -kIntMagic), s_lo * unit.x, acc[a][0]);
              acc[a][1] = fmaf(__uint_as_float(d[1]) + fmaf(-z_lo, sum.y, -kIntMagic), s_lo * unit.y, acc[a][1]);
              acc[a][2] = fmaf(__uint_as_float(d[2]) + fmaf(-z_hi, sum.x, -kIntMagic), s_hi * unit.x, acc[a][2]);
              acc[a][3] = fmaf(__uint_as_float(d[3]) + fmaf(-z_hi, sum.y, -kIntMagic), s_hi * unit.y, acc[a][3]);
            }
          }
        }
      }
      // by the lanes t = 0 and t = 2, which hold the first digits of token 0 and of token 1
      const uint32_t marked = __ballot_sync(0xffffffffu, unit.x == 0.0f) & (tokens == 1 ? 1u : 5u);
      if (marked) {
        const unsigned char* token = digits + (p - slab) * (4 * kDigitCols * 64);
#pragma unroll
        for (int a = 0; a < MATS; ++a) {
          const float2 add = span_products<T, GROUPS>(ring + take + a * C::SLOT + (place[a] & 127u), w[a].zeros != 0, token,
                                                      min(2, s.col_tiles - 2 * p), marked);
          acc[a][0] = fmaf(add.x, 1.0f / H::kUnit, acc[a][0]);
          acc[a][2] = fmaf(add.y, 1.0f / H::kUnit, acc[a][2]);
        }
      }
      take = take == (DEPTH - 1) * C::PAIR ? 0 : take + C::PAIR;
#pragma unroll
      for (int a = 0; a < MATS; ++a) place[a] += 2 * COL_WARPS * block_bytes(GROUPS, w[a].zeros);
    }
  }

  copies_wait<0>();
  // A token's columns, added up: with two tokens one has the lanes t = 0 and 1 and the other t = 2 and 3, with one it has all.
  const uint32_t arrivals = smem_addr + C::RING + C::DIGITS + C::SUMS + C::UNITS;
  float* leaving = reinterpret_cast<float*>(smem + warp * (DEPTH * C::PAIR));  // [matrix][token][row] of this warp
#pragma unroll
  for (int a = 0; a < MATS; ++a)
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const float own = acc[a][2 * hi] + acc[a][2 * hi + 1], four = own + __shfl_down_sync(0xffffffffu, own, 1);
      const float eight = four + __shfl_down_sync(0xffffffffu, four, 2);
      if (t % 2 == 0 && t / 2 < tokens)
        leaving[(a * kDigitTokens + t / 2) * kTileRows + g + 8 * hi] = tokens == 1 ? eight : four;
    }
  __syncwarp();
  cluster_wait();
  if (lane < MATS * kDigitTokens * 4) {
    const int a = lane / (kDigitTokens * 4), tok = lane / 4 % kDigitTokens;
    const int o = tok * kRows + row_warp * kTileRows + lane % 4 * 4, owner = (int)((unsigned)o / (unsigned)slice);
    if (tok < tokens)
      cluster_send4(arrivals + ((a * COL_WARPS + col_warp) * (C::OUTPUTS + 64) + rank * slice + o - owner * slice) * 4,
                    tc::smem_u32(sums), owner, *reinterpret_cast<const float4*>(leaving + lane * 4));
  }
  const bool there_in_time = mine <= 0 || own_wait(sums, 0);
  const float* parts = reinterpret_cast<const float*>(smem + C::RING + C::DIGITS + C::SUMS + C::UNITS);
  const int begin = rank * slice, o = threadIdx.x;  // mine <= OUTPUTS <= 32 * kWarps
  const int row = (begin + o) % kRows, tok = (begin + o) / kRows;
  const long long n = (long long)row_tile0 * kTileRows + row;
  if (o < mine && n < s.n) {
    float v[MATS];
#pragma unroll
    for (int a = 0; a < MATS; ++a) {
      v[a] = 0.0f;
#pragma unroll 1
      for (int i = 0; i < split; ++i)
#pragma unroll
        for (int q = 0; q < COL_WARPS; ++q) v[a] += parts[(a * COL_WARPS + q) * (C::OUTPUTS + 64) + i * slice + o];
    }
    if (!there_in_time) v[0] = __uint_as_float(0x7fffffffu);
    const Consts consts(gm, dm);
    static_cast<uint16_t*>(y)[tok * s.y_pitch + n] = H::from_float(result<MATS>(v, activation, consts));
  }
}

// ------------------------------------------------------------------ written out

// A lane's words of block (row_tile, c): for u = 0..3 and both rows, eight numbers, handed to `put(hi, u, v)`.
template <class T, class F>
__device__ __forceinline__ void dequantize_block(const W4& w, const W4Shape& s, long long row_tile, int c, F&& put) {
  using H = Half2<T>;
  const int lane = threadIdx.x & 31, g = lane >> 2, groups = 1 << s.groups_log2;
  const char* block = cbyte(w.blocks) + (row_tile * s.col_tiles + c) * block_bytes(groups, w.zeros);
  const Vec<16> q[2] = {Ld<16, LD_NC_NOALLOC>::ld(block + lane * 16), Ld<16, LD_NC_NOALLOC>::ld(block + 512 + lane * 16)};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int at = (g * groups + (u >> (2 - s.groups_log2))) * 2;
    const uint32_t sc = Ld<4, LD_PLAIN>::ld(block + kTileBytes + at * 2).w[0];
    const uint32_t z = w.zeros ? Ld<2, LD_PLAIN>::ld(block + kTileBytes + groups * 32 + at).w[0] : 0x0808u;
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const float scale = H::to_float(hi ? sc >> 16 : sc & 0xffffu);
      const float zero = __uint_as_float(0x4b000000u | (hi ? z >> 8 : z & 0xffu));  // 2^23 + z, and the code 2^23 + q
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        f[e] = (__uint_as_float((q[hi].w[u] >> (2 * e + 14 * (e & 1)) & 15u) | 0x4b000000u) - zero) * scale;
      Vec<16> v;
      Codec<T>::template pack<16>(f, v);  // the one rounding
      put(hi, u, v);
    }
  }
}

// Rows that start on 16-byte boundaries and end in whole pieces of 8 columns: a warp per block, every lane stores its
// pieces where they belong, 64 bytes of a row at a time.
template <class T>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(void* out, W4 w, W4Shape s) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long tile = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), row_tile = tile / s.col_tiles;
  const int c = (int)(tile - row_tile * s.col_tiles);
  if (row_tile * kTileRows >= s.n) return;
  dequantize_block<T>(w, s, row_tile, c, [&](int hi, int u, const Vec<16>& v) {
    const long long row = row_tile * kTileRows + 8 * hi + g, k = (long long)c * kTileCols + 32 * u + 8 * t;
    if (row < s.n && k < s.k) St<16, ST_CS>::st(byte(out) + (row * s.y_pitch + k) * 2, v);
  });
}

// Any other rows.  A CTA writes 16 rows x 512 columns: each warp turns one block into numbers in shared memory, then the
// warps write the rows, a 32-byte frame a lane, through the realigned stores of swiglu_kernels.cuh.
constexpr int kOutTiles = 4, kOutPitch = kOutTiles * kTokenBytes + 64;  // this pitch keeps a warp's stores on different banks

template <class T>
__global__ void __launch_bounds__(32 * kOutTiles) w4_dequantize_rows_kernel(void* out, W4 w, W4Shape s) {
  __shared__ __align__(16) unsigned char rows[kTileRows * kOutPitch];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long row_tile = (long long)blockIdx.y + (long long)blockIdx.z * gridDim.y;
  if (row_tile * kTileRows >= s.n) return;
  const int c = (int)blockIdx.x * kOutTiles + warp;
  if (c < s.col_tiles)
    dequantize_block<T>(w, s, row_tile, c, [&](int hi, int u, const Vec<16>& v) {
      *reinterpret_cast<Vec<16>*>(rows + (8 * hi + g) * kOutPitch + warp * kTokenBytes + (32 * u + 8 * t) * 2) = v;
    });
  __syncthreads();
  const long long k = (long long)blockIdx.x * (kOutTiles * kTileCols) + lane * 16, left = s.k - k;
#pragma unroll 1
  for (int r = warp; r < kTileRows && row_tile * kTileRows + r < s.n; r += kOutTiles) {
    const Vec<16>* from = reinterpret_cast<const Vec<16>*>(rows + r * kOutPitch + lane * 32);
    const Vec<16> a = from[0], b = from[1];
    const Vec<32> v = {{a.w[0], a.w[1], a.w[2], a.w[3], b.w[0], b.w[1], b.w[2], b.w[3]}};
    char* dst = byte(out) + ((row_tile * kTileRows + r) * s.y_pitch + k) * 2;
    st_skewed32<ST_CS>(dst, v, (int)((uintptr_t)dst & 31), left >= 16, lane == 0, lane == 31 || left < 32);
    if (left > 0 && left < 16) {
#pragma unroll
      for (int e = 0; e < 15; ++e)
        if (e < left) {
          Vec<2> o;
          o.w[0] = v.w[e / 2] >> (16 * (e & 1)) & 0xffffu;
          St<2, ST_PLAIN>::st(dst + 2 * e, o);
        }
    }
  }
}

// ------------------------------------------------------------------ host side

constexpr long long kMaxSize = 1LL << 30;  // of n and k: tile counts and copies' coordinates fit an int, byte offsets 62 bits

// Checks shared by the three entries; fills the shape.
int check(const W4* w, int mats, int64_t n, int64_t k, int group, int dtype, W4Shape& s) {
  if (dtype != SWIGLU_B200_F16 && dtype != SWIGLU_B200_BF16) return SWIGLU_B200_ERR_DTYPE;
  if (group != 32 && group != 64 && group != 128) return SWIGLU_B200_ERR_ARG;
  if (n < 0 || k < 0 || n > kMaxSize || k > kMaxSize) return SWIGLU_B200_ERR_SHAPE;
  if (n > 0 && k > 0 && n > (1LL << 60) / k) return SWIGLU_B200_ERR_SHAPE;
  s.n = n;
  s.k = k;
  const long long col_tiles = (k + kTileCols - 1) / kTileCols;
  if (col_tiles > 0x7fffffffLL / 4) return SWIGLU_B200_ERR_SHAPE;
  s.col_tiles = (int)col_tiles;
  s.groups_log2 = group == 128 ? 0 : group == 64 ? 1 : 2;
  for (int i = 0; i < mats; ++i) {
    if (n == 0 || k == 0) break;
    if (!w[i].blocks) return SWIGLU_B200_ERR_NULL;
    if (address(w[i].blocks) % 16) return SWIGLU_B200_ERR_ALIGN;
  }
  return SWIGLU_B200_OK;
}

// The bytes that a call reads of one matrix.
ByteRange weight_range(const W4& w, const W4Shape& s) {
  const long long tiles = (s.n + kTileRows - 1) / kTileRows * s.col_tiles;
  return byte_range(w.blocks, 1, tiles * block_bytes(1 << s.groups_log2, w.zeros), 0);
}

// What is known of a kernel on each device: whether its limit of shared memory has been raised, and how many clusters of
// each size run at once (0: not asked yet).  Written once per device and size; every writer writes the same.
struct Launcher {
  std::atomic<uint64_t> opted_in{0};
  std::atomic<int> clusters[64][9] = {};
};

template <class X> using Kernel = void (*)(void*, X, W4, W4, W4Shape, int, float, float);

// One of the kernels above on the current device.
template <class X> struct Start {
  Kernel<X> kernel;
  Launcher& known;
  int threads, smem, device = 0;
  cudaLaunchAttribute attrs[2] = {};
  cudaLaunchConfig_t cfg{};

  Start(Kernel<X> kernel, Launcher& known, int threads, int smem)
      : kernel(kernel), known(known), threads(threads), smem(smem) {}

  int prepare(cudaStream_t st) {
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && !(device < 64 && (known.opted_in.load(std::memory_order_relaxed) >> device & 1))) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e == cudaSuccess && device < 64) known.opted_in.fetch_or(1ULL << device, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_DEVICE, e);
    attrs[0].id = cudaLaunchAttributeClusterDimension;
    attrs[0].val.clusterDim.y = attrs[0].val.clusterDim.z = 1;
    attrs[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cfg.attrs = attrs;
    return SWIGLU_B200_OK;
  }
  // How many clusters of `split` CTAs run at once, with a few places left free (with every one taken 1 x 8192 -> 3584 took
  // 7.3 us, not 5.4); negative: an error code.
  int at_once(int split) {
    int n = device < 64 ? known.clusters[device][split].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
      attrs[0].val.clusterDim.x = (unsigned)split;
      cfg.gridDim = dim3((unsigned)split);
      cfg.numAttrs = 1;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
      if (e != cudaSuccess) return -note_cuda_error(SWIGLU_B200_ERR_DEVICE, e);
      if (device < 64) known.clusters[device][split].store(n, std::memory_order_relaxed);
    }
    return n - n / 32;
  }
  int launch(long long clusters, long long gy, void* y, const X& x, const W4* w, int mats, const W4Shape& s, int activation,
             float gm, float dm) {
    attrs[0].val.clusterDim.x = (unsigned)s.split;
    cfg.gridDim = dim3((unsigned)(clusters * s.split), (unsigned)gy);
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, y, x, w[0], w[mats - 1], s, activation, gm, dm);
    if (e != cudaSuccess) {
      cudaGetLastError();
      return note_cuda_error(SWIGLU_B200_ERR_LAUNCH, e);
    }
    note_launch();
    return SWIGLU_B200_OK;
  }
};

// Launches `kernel` with `clusters` clusters.  Its `parts` column tiles (or pairs) are split over
// the CTAs of a cluster, as many as leave every cluster running at once: all of them stream from the start and end
// together (one cluster more than fit is another round, 430 CTAs instead of 258 took 22.8 us instead of 19.9).
// `outputs` are a cluster's, finished in slices of a multiple of `unit`.
int start(Kernel<const void*> kernel, Launcher& known, long long clusters, int parts, int outputs, int unit, int smem,
          cudaStream_t st, void* y, const void* x, const W4* w, int mats, W4Shape s, int activation, float gm,
          float dm) {
  if (clusters > 0x7fffffffLL / 8) return SWIGLU_B200_ERR_SHAPE;
  Start<const void*> k(kernel, known, 32 * kWarps, smem);
  int rc = k.prepare(st);
  if (rc != SWIGLU_B200_OK) return rc;
  int split = parts < 8 ? parts : 8;
  for (; split > 1; --split) {
    const int at_once = k.at_once(split);
    if (at_once < 0) return -at_once;
    if (clusters <= at_once) break;
  }
  s.split = split;
  s.share = parts / split;
  s.over = parts % split;
  s.slice = (outputs + unit * split - 1) / (unit * split) * unit;
  return k.launch(clusters, 1, y, x, w, mats, s, activation, gm, dm);
}

template <class T, int MATS, int NT, int GROUPS>
int launch(void* y, const void* x, const W4* w, const W4Shape& s, int activation, float gm, float dm, cudaStream_t st) {
  constexpr int kRows = kWarps * kTileRows;
  static Launcher known;
  return start(w4_kernel<T, MATS, NT, GROUPS>, known, (s.n + kRows - 1) / kRows, s.col_tiles, kRows * (int)s.m, 4,
               Cfg<MATS, NT, GROUPS>::SMEM, st, y, x, w, MATS, s, activation, gm, dm);
}

template <class T, int MATS, int N, int GROUPS>
int launch_mma(void* y, const void* x, const W4* w, const W4Shape& s, int activation, float gm, float dm, cudaStream_t st) {
  static Launcher known;
  const tc::EncodeTiled encode = tc::encode_fn();
  if (!encode) return SWIGLU_B200_ERR_DEVICE;
  Maps maps;
  const cuuint32_t steps[2] = {1, 1};
  const cuuint64_t x_dims[2] = {(cuuint64_t)s.k, (cuuint64_t)s.m}, x_pitch[1] = {(cuuint64_t)s.x_pitch * 2};
  const cuuint32_t x_box[2] = {64, N};
  bool mapped = encode(&maps.x, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(x), x_dims, x_pitch, x_box, steps,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  for (int a = 0; a < MATS && mapped; ++a) {
    const cuuint64_t pitch[1] = {(cuuint64_t)s.col_tiles * block_bytes(GROUPS, w[a].zeros)};
    const cuuint64_t dims[2] = {pitch[0] / 8, (cuuint64_t)((s.n + kTileRows - 1) / kTileRows)};
    const cuuint32_t box[2] = {(cuuint32_t)slot_bytes(GROUPS, w[a].zeros) / 8, kGroupRows / kTileRows};
    mapped = encode(&maps.w[a], CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<void*>(w[a].blocks), dims, pitch, box, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
  if (!mapped) return SWIGLU_B200_ERR_DEVICE;
  Start<Maps> k(w4_mma_kernel<T, MATS, N, GROUPS>, known, kGroups * kGroupThreads, MmaCfg<N, GROUPS>::SMEM);
  int rc = k.prepare(st);
  if (rc != SWIGLU_B200_OK) return rc;
  const long long row_groups = (s.n + kGroupRows - 1) / kGroupRows, gy = (s.m + N - 1) / N;
  if (row_groups > 0x7fffffffLL / 8 || gy > 65535) return SWIGLU_B200_ERR_SHAPE;
  // The fewest column tiles to a warpgroup with every cluster running at once: gate and up of 4096 -> 11008 have 86 groups
  // of 128 rows, two to each of 43 clusters of three CTAs are 11 tiles to a warpgroup, one to each of 86 CTAs 16.
  int best = 0, split = 1, groups = 1;
  for (int r = 1; r <= 4; ++r)
    for (int c = 1; c <= 8; ++c) {
      if (kGroups * c % (r * MATS)) continue;
      const int parts = kGroups * c / (r * MATS), cost = (s.col_tiles + parts - 1) / parts;
      if (best != 0 && cost >= best) continue;
      const int at_once = k.at_once(c);
      if (at_once < 0) return -at_once;
      if ((row_groups + r - 1) / r * gy <= at_once) best = cost, split = c, groups = r;
    }
  W4Shape shape = s;
  shape.split = split;
  shape.row_groups = groups;
  shape.slice = (groups * (int)(s.m < N ? s.m : N) + split - 1) / split;
  return k.launch((row_groups + groups - 1) / groups, gy, y, maps, w, MATS, shape, activation, gm, dm);
}

template <class T, int MATS, int GROUPS, int ROW_WARPS>
int launch_digits(void* y, const void* x, const W4* w, const W4Shape& s, int activation, float gm, float dm,
                  cudaStream_t st) {
  constexpr int kRows = ROW_WARPS * kTileRows;
  static Launcher known;
  return start(w4_digits_kernel<T, MATS, GROUPS, ROW_WARPS>, known, (s.n + kRows - 1) / kRows, (s.col_tiles + 1) / 2,
               kRows * (int)s.m, 4, DigitCfg<MATS, GROUPS, ROW_WARPS>::SMEM, st, y, x, w, MATS, s, activation, gm, dm);
}

constexpr int kEnoughCtas = 192;  // one to a SM and some more

template <int MATS>
int run(void* y, const void* x, const W4* w, W4Shape s, int64_t m, int64_t x_row_stride, int64_t y_row_stride,
        int dtype, int activation, float gm, float dm, int device, void* stream) {
  if (m < 0) return SWIGLU_B200_ERR_SHAPE;
  if (m == 0 || s.n == 0) return SWIGLU_B200_OK;
  if (s.k == 0) return SWIGLU_B200_ERR_SHAPE;
  if (x_row_stride < s.k || y_row_stride < s.n) return SWIGLU_B200_ERR_SHAPE;
  if (!fits_address_space(m, x_row_stride, 2) || !fits_address_space(m, y_row_stride, 2)) return SWIGLU_B200_ERR_SHAPE;
  if (!y || !x) return SWIGLU_B200_ERR_NULL;
  if (address(y) % 2 || address(x) % 16 || (m > 1 && x_row_stride % 8)) return SWIGLU_B200_ERR_ALIGN;
  const ByteRange out = byte_range(y, m, s.n * 2, y_row_stride * 2);
  if (overlap(out, byte_range(x, m, s.k * 2, x_row_stride * 2))) return SWIGLU_B200_ERR_ALIAS;
  for (int i = 0; i < MATS; ++i)
    if (overlap(out, weight_range(w[i], s))) return SWIGLU_B200_ERR_ALIAS;
  CallDevice scope(device);
  if (scope.err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_DEVICE, scope.err);
  s.m = m;
  s.x_pitch = x_row_stride;
  s.y_pitch = y_row_stride;
  s.y_vec = address(y) % 8 == 0 && y_row_stride % 4 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto typed = [&](auto t) {
    using T = decltype(t);
    auto grouped = [&](auto groups) {
      constexpr int G = decltype(groups)::value;
      if (m <= kDigitTokens) {
        // 128 rows to a CTA leave it a shorter part of the tokens to make digits of, and can be split more evenly; 64 rows
        // make more CTAs where there are few rows, and smaller clusters (us, 64 and 128: 5000 -> 6000 6.9 and 5.5, 6144 -> 4096
        // 4.9 and 4.8, 2048 -> 4096 3.0 and 3.2, 8192 -> 2048 4.1 and 5.3, gate and up 4096 -> 11008 13.2 and 10.7, 2048 -> 5504
        // 4.5 and 5.0).  Of 18 shapes between 1024 -> 2048 and 4096 -> 11008 the other side was faster by more than 2 % in two,
        // gate and up 4096 -> 4096 (5.2 against 5.7) and 2048 -> 2048 (3.7 against 4.0).
        const long long pairs = (s.col_tiles + 1) / 2;
        if (pairs >= 16 && (s.n + 127) / 128 * 8 >= kEnoughCtas)
          return launch_digits<T, MATS, G, 8>(y, x, w, s, activation, gm, dm, st);
        return launch_digits<T, MATS, G, 4>(y, x, w, s, activation, gm, dm, st);
      }
      // A launch of w4_mma_kernel starts and ends about 1 us slower, one of w4_kernel takes longer for each weight and 8 tokens
      // (us, w4_kernel and w4_mma_kernel: 4096 -> 4096 with 8 tokens 4.6 and 6.2, with 32 7.6 and 8.4, with 64 12.1 and 11.9;
      // 14336 -> 4096 with 8 tokens 11.2 and 11.3, with 16 13.0 and 11.8, with 32 19.3 and 13.3): lines through these times
      // cross at this many weights.  Of 48 cases in fp16 from 4 to 32 tokens and 2048 -> 4096 to 4096 -> 11008 the other side was
      // faster by more than 4 % in five: 20 tokens 4096 -> 6144 (9.1 against 10.2) and gate and up of 2048 and 2731 square with
      // 20 and 32 (5 to 9 %).
      if (m > 32 || ((double)s.n * (double)s.k * MATS - 0x1p24) * (double)((m + 7) / 8 * 8) >= 0x1p28) {
        if (m <= 16) return launch_mma<T, MATS, 16, G>(y, x, w, s, activation, gm, dm, st);
        if (m <= 32) return launch_mma<T, MATS, 32, G>(y, x, w, s, activation, gm, dm, st);
        return launch_mma<T, MATS, 64, G>(y, x, w, s, activation, gm, dm, st);
      }
      if (m <= 8) return launch<T, MATS, 1, G>(y, x, w, s, activation, gm, dm, st);
      if (m <= 16) return launch<T, MATS, 2, G>(y, x, w, s, activation, gm, dm, st);
      if (m <= 24) return launch<T, MATS, 3, G>(y, x, w, s, activation, gm, dm, st);
      return launch<T, MATS, 4, G>(y, x, w, s, activation, gm, dm, st);
    };
    if (s.groups_log2 == 0) return grouped(std::integral_constant<int, 1>{});
    if (s.groups_log2 == 1) return grouped(std::integral_constant<int, 2>{});
    return grouped(std::integral_constant<int, 4>{});
  };
  return dtype == SWIGLU_B200_F16 ? typed(__half{}) : typed(__nv_bfloat16{});
}

}  // namespace

extern "C" {

int swiglu_b200_w4_linear(void* y, const void* x, const void* blocks, int zeros, int64_t m, int64_t n, int64_t k,
                          int64_t x_row_stride, int64_t y_row_stride, int group, int dtype, int device, void* stream) {
  const W4 w{blocks, zeros != 0};
  W4Shape s{};
  const int rc = check(&w, 1, n, k, group, dtype, s);
  if (rc != SWIGLU_B200_OK) return rc;
  return run<1>(y, x, &w, s, m, x_row_stride, y_row_stride, dtype, SWIGLU_B200_SILU, 1.0f, 1.0f, device, stream);
}

int swiglu_b200_w4_gate_up(void* h, const void* x, const void* gate_blocks, int gate_zeros, const void* up_blocks,
                           int up_zeros, int64_t m, int64_t n, int64_t k, int64_t x_row_stride, int64_t h_row_stride,
                           int group, int dtype, int activation, float gm, float dm, int device, void* stream) {
  const W4 w[2] = {{gate_blocks, gate_zeros != 0}, {up_blocks, up_zeros != 0}};
  W4Shape s{};
  const int rc = check(w, 2, n, k, group, dtype, s);
  if (rc != SWIGLU_B200_OK) return rc;
  if (activation < SWIGLU_B200_SILU || activation > SWIGLU_B200_GELU_ERF) return SWIGLU_B200_ERR_ARG;
  return run<2>(h, x, w, s, m, x_row_stride, h_row_stride, dtype, activation, gm, dm, device, stream);
}

int swiglu_b200_w4_dequantize(void* out, const void* blocks, int zeros, int64_t n, int64_t k, int64_t out_row_stride,
                              int group, int dtype, int device, void* stream) {
  const W4 w{blocks, zeros != 0};
  W4Shape s{};
  const int rc = check(&w, 1, n, k, group, dtype, s);
  if (rc != SWIGLU_B200_OK) return rc;
  if (n == 0 || k == 0) return SWIGLU_B200_OK;
  if (out_row_stride < k || !fits_address_space(n, out_row_stride, 2)) return SWIGLU_B200_ERR_SHAPE;
  if (!out) return SWIGLU_B200_ERR_NULL;
  if (address(out) % 2) return SWIGLU_B200_ERR_ALIGN;
  const ByteRange o = byte_range(out, n, k * 2, out_row_stride * 2);
  if (overlap(o, weight_range(w, s))) return SWIGLU_B200_ERR_ALIAS;
  const long long row_tiles = (n + kTileRows - 1) / kTileRows;
  CallDevice scope(device);
  if (scope.err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_DEVICE, scope.err);
  s.y_pitch = out_row_stride;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto typed = [&](auto t) {
    using T = decltype(t);
    // fp16 5504 x 2096: 6.7 us stored directly, 9.6 us through shared memory; 5503 x 2091, where the direct form would
    // store element by element, 51.9 and 12.5 us
    const long long ctas = (row_tiles * s.col_tiles + 7) / 8;
    if (address(out) % 16 == 0 && out_row_stride % 8 == 0 && k % 8 == 0 && ctas <= 0x7fffffffLL) {
      w4_dequantize_kernel<T><<<(unsigned)ctas, 256, 0, st>>>(out, w, s);
    } else {
      const long long z = (row_tiles + 65534) / 65535, y = (row_tiles + z - 1) / z;
      w4_dequantize_rows_kernel<T><<<dim3((unsigned)((s.col_tiles + kOutTiles - 1) / kOutTiles), (unsigned)y, (unsigned)z),
                                     32 * kOutTiles, 0, st>>>(out, w, s);
    }
  };
  dtype == SWIGLU_B200_F16 ? typed(__half{}) : typed(__nv_bfloat16{});
  return launched();
}

}  // extern "C"
