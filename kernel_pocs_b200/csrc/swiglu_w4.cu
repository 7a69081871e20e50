// Projections with 4-bit weights and group scales for a few tokens (declarations: include/swiglu_b200.h):
//
//   y[m][n] = sum_k x[m][k] * (q[n][k] - z[n][k/G]) * s[n][k/G]            q in 0..15, G = 32, 64 or 128
//   h[m][n] = act(gm * (x . w_gate[n])) * (x . w_up[n]) * dm               both projections in one launch
//
// With a handful of tokens the weights' bytes are the whole cost (n*k/2, each used 2m times), so the kernels are
// streams of weights with as little arithmetic per weight as it takes.  The products go through mma.sync m16n8k16: 16
// weight rows are the A operand, 8 tokens the B operand, accumulation in fp32.  The tensor pipe is far from busy here;
// what the instruction saves is issue slots (one weight per lane and FMA would need 8 m of them for 8 weights).  Eight
// nibbles become four pairs of 16-bit numbers with a mask, an OR that puts them into the mantissa of 128 (bf16) or 1024
// (fp16), and an exact subtraction of that plus the zero point.  q - z is exact in either type; the sum over a group is
// a fp32 accumulator which is multiplied by the group's scale in fp32: nothing is rounded to 16 bits before the result.
//
// Weight tiles.  The fragments fix which lane needs which nibbles, so weights are laid out once for it: 16 rows x 128
// columns are 1 KB in which lane l = 4g + t finds the 32 nibbles of row g (and, 512 bytes on, of row g + 8) that it
// feeds to the tile's eight instructions, as one 16-byte load; a warp's load is 512 contiguous bytes and the tiles of a
// row are contiguous along k.  Word u of a lane holds columns 32u + 8t .. +7, so the 4 lanes of a row cover 32 columns
// with each word and a group of 32 never mixes with the next inside one instruction.
#include "swiglu_b200.h"

#include <type_traits>

#include "launch_common.cuh"
#include "swiglu_kernels.cuh"

namespace {

using namespace swiglu_b200;

constexpr int kTileRows = 16, kTileCols = 128, kTileBytes = kTileRows * kTileCols / 2;
constexpr int kWarps = 8;

// One 4-bit weight matrix in tiles.
struct W4 {
  const void* tiles;   // [row tiles][column tiles][2][32][16 bytes]
  const void* scales;  // [row tiles][groups][8][2], rows g and g + 8 side by side
  const void* zeros;   // uint8, laid out as the scales; NULL means 8 everywhere
};

struct W4Shape {
  long long m, n, k;
  long long x_pitch, y_pitch;  // elements
  int col_tiles;
  int groups_log2;  // log2 of the groups per column tile (0, 1, 2)
  int x_vec;        // every row of x starts on a 16-byte boundary
};

template <class T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
  using V = __nv_bfloat162;
  static constexpr uint32_t kMagic = 0x43004300u;  // (128, 128): one step of the mantissa is 1
  static __device__ __forceinline__ uint32_t magic_plus(uint32_t z) { return kMagic + z * 0x00010001u; }
  static __device__ __forceinline__ float to_float(uint32_t half_word) { return __uint_as_float(half_word << 16); }
  static __device__ __forceinline__ uint16_t from_float(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Half2<__half> {
  using V = __half2;
  static constexpr uint32_t kMagic = 0x64006400u;  // (1024, 1024)
  static __device__ __forceinline__ uint32_t magic_plus(uint32_t z) { return kMagic + z * 0x00010001u; }
  static __device__ __forceinline__ float to_float(uint32_t half_word) {
    return __half2float(__ushort_as_half((unsigned short)half_word));
  }
  static __device__ __forceinline__ uint16_t from_float(float f) { return __half_as_ushort(__float2half_rn(f)); }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Nibbles I and I + 4 of a word as a pair of exact 16-bit numbers q - z.
template <class T, int I>
__device__ __forceinline__ uint32_t weight_pair(uint32_t word, uint32_t bias) {
  using V = typename Half2<T>::V;
  uint32_t w = ((word >> (4 * I)) & 0x000f000fu) | Half2<T>::kMagic;
  V r = __hsub2(*reinterpret_cast<V*>(&w), *reinterpret_cast<V*>(&bias));
  return *reinterpret_cast<uint32_t*>(&r);
}

// Columns k .. k+7 of a row of x, zero past column K.
template <class T>
__device__ __forceinline__ Vec<16> x_load(const char* row, long long k, long long K, bool vec) {
  if (vec && k + 8 <= K) return Ld<16, LD_PLAIN>::ld(row + k * 2);
  Vec<16> v{};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < K) v.w[e / 2] |= Ld<2, LD_PLAIN>::ld(row + (k + e) * 2).w[0] << (16 * (e & 1));
  return v;
}

// A CTA owns RT row tiles of MATS matrices and NT * 8 tokens; its warps share the column tiles among them and add
// their sums up in shared memory.
template <class T, int MATS, int RT, int NT, int ACT>
__global__ void __launch_bounds__(32 * kWarps)
w4_kernel(void* y, const void* __restrict__ x, W4 w0, W4 w1, W4Shape s, float gm, float dm) {
  using H = Half2<T>;
  __shared__ float red[kWarps][MATS * RT * NT * 4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long row_tile = (long long)blockIdx.x * RT, row_tiles = (s.n + kTileRows - 1) / kTileRows;
  const long long token0 = (long long)blockIdx.y * (8 * NT);
  const W4 w[2] = {w0, w1};

  float acc[MATS][RT][NT][4] = {};
  for (int c = warp; c < s.col_tiles; c += kWarps) {
    Vec<16> q[MATS][RT][2];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const bool there = row_tile + r < row_tiles;
        const char* p = cbyte(w[i].tiles) + ((row_tile + r) * s.col_tiles + c) * kTileBytes + lane * 16;
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) q[i][r][hi] = there ? Ld<16, LD_NC_NOALLOC>::ld(p + hi * 512) : Vec<16>{};
      }
    Vec<16> b[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const long long token = token0 + j * 8 + g;
      const char* row = cbyte(x) + token * s.x_pitch * 2;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        b[j][u] = token < s.m ? x_load<T>(row, (long long)c * kTileCols + 32 * u + 8 * t, s.k, s.x_vec) : Vec<16>{};
    }
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (row_tile + r >= row_tiles) continue;
        const long long group0 = ((row_tile + r) * s.col_tiles + c) << s.groups_log2;
        float part[NT][4] = {};
        uint32_t bias_lo = 0, bias_hi = 0;
        float scale_lo = 0, scale_hi = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int per_group = 4 >> s.groups_log2;  // words per group
          if (u % per_group == 0) {
            const long long at = (group0 + u / per_group) * 16 + 2 * g;
            const uint32_t sc = Ld<4, LD_PLAIN>::ld(cbyte(w[i].scales) + at * 2).w[0];
            scale_lo = H::to_float(sc & 0xffffu);
            scale_hi = H::to_float(sc >> 16);
            const uint32_t z = w[i].zeros ? Ld<2, LD_PLAIN>::ld(cbyte(w[i].zeros) + at).w[0] : 0x0808u;
            bias_lo = H::magic_plus(z & 0xffu);
            bias_hi = H::magic_plus(z >> 8);
          }
          const uint32_t lo = q[i][r][0].w[u], hi = q[i][r][1].w[u];
          const uint32_t a0[4] = {weight_pair<T, 0>(lo, bias_lo), weight_pair<T, 0>(hi, bias_hi),
                                  weight_pair<T, 1>(lo, bias_lo), weight_pair<T, 1>(hi, bias_hi)};
          const uint32_t a1[4] = {weight_pair<T, 2>(lo, bias_lo), weight_pair<T, 2>(hi, bias_hi),
                                  weight_pair<T, 3>(lo, bias_lo), weight_pair<T, 3>(hi, bias_hi)};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint32_t* xw = b[j][u].w;  // columns (0,1) (2,3) (4,5) (6,7) of the lane's eight
            H::mma(part[j], a0, __byte_perm(xw[0], xw[2], 0x5410), __byte_perm(xw[0], xw[2], 0x7632));
            H::mma(part[j], a1, __byte_perm(xw[1], xw[3], 0x5410), __byte_perm(xw[1], xw[3], 0x7632));
          }
          if ((u + 1) % per_group == 0) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              acc[i][r][j][0] = fmaf(part[j][0], scale_lo, acc[i][r][j][0]);
              acc[i][r][j][1] = fmaf(part[j][1], scale_lo, acc[i][r][j][1]);
              acc[i][r][j][2] = fmaf(part[j][2], scale_hi, acc[i][r][j][2]);
              acc[i][r][j][3] = fmaf(part[j][3], scale_hi, acc[i][r][j][3]);
              part[j][0] = part[j][1] = part[j][2] = part[j][3] = 0.0f;
            }
          }
        }
      }
  }

#pragma unroll
  for (int i = 0; i < MATS; ++i)
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][((i * RT + r) * NT + j) * 4 + e][lane] = acc[i][r][j][e];
  __syncthreads();

  const Consts consts(gm, dm);
  for (int o = threadIdx.x; o < RT * kTileRows * NT * 8; o += 32 * kWarps) {
    const int row = o % (RT * kTileRows), tok = o / (RT * kTileRows);
    const long long n = row_tile * kTileRows + row, token = token0 + tok;
    if (n >= s.n || token >= s.m) continue;
    // where lane 4g + t keeps (row g + 8 hi, token 2t + lo) of a tile
    const int r = row / kTileRows, hi = row / 8 % 2, slot = (row % 8) * 4 + tok % 8 / 2;
    float v[MATS];
#pragma unroll
    for (int i = 0; i < MATS; ++i) {
      const int at = ((i * RT + r) * NT + tok / 8) * 4 + 2 * hi + tok % 2;
      v[i] = 0.0f;
#pragma unroll
      for (int p = 0; p < kWarps; ++p) v[i] += red[p][at][slot];
    }
    float out = v[0];
    if constexpr (MATS == 2) out = Math<true, ACT>::fwd(v[0], v[1], consts);
    static_cast<uint16_t*>(y)[token * s.y_pitch + n] = H::from_float(out);
  }
}

// One warp per tile: every lane writes four runs of 8 columns in each of its two rows.
template <class T>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(void* out, W4 w, W4Shape s, int out_vec) {
  using H = Half2<T>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long tile = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const long long row_tile = tile / s.col_tiles;
  const int c = (int)(tile - row_tile * s.col_tiles);
  if (row_tile * kTileRows >= s.n) return;
  const char* p = cbyte(w.tiles) + tile * kTileBytes + lane * 16;
  const Vec<16> q[2] = {Ld<16, LD_NC_NOALLOC>::ld(p), Ld<16, LD_NC_NOALLOC>::ld(p + 512)};
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const long long at = ((tile << s.groups_log2) + (u >> (2 - s.groups_log2))) * 16 + 2 * g;
    const uint32_t sc = Ld<4, LD_PLAIN>::ld(cbyte(w.scales) + at * 2).w[0];
    const uint32_t z = w.zeros ? Ld<2, LD_PLAIN>::ld(cbyte(w.zeros) + at).w[0] : 0x0808u;
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const long long row = row_tile * kTileRows + 8 * hi + g;
      const long long k = (long long)c * kTileCols + 32 * u + 8 * t;
      if (row >= s.n || k >= s.k) continue;
      const float scale = H::to_float(hi ? sc >> 16 : sc & 0xffffu);
      const int zero = hi ? z >> 8 : z & 0xff;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)((int)(q[hi].w[u] >> (4 * e) & 15u) - zero) * scale;
      Vec<16> v;
      Codec<T>::template pack<16>(f, v);
      char* dst = byte(out) + (row * s.y_pitch + k) * 2;
      if (out_vec && k + 8 <= s.k) {
        St<16, ST_PLAIN>::st(dst, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < s.k) {
            Vec<2> o;
            o.w[0] = v.w[e / 2] >> (16 * (e & 1)) & 0xffffu;
            St<2, ST_PLAIN>::st(dst + 2 * e, o);
          }
      }
    }
  }
}

// ------------------------------------------------------------------ host side

int launched() {
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_LAUNCH, err);
  note_launch();
  return SWIGLU_B200_OK;
}

constexpr long long kMaxSize = 1LL << 40;  // of n and k: tile counts and byte offsets stay within 62 bits

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
    if (!w[i].tiles || !w[i].scales) return SWIGLU_B200_ERR_NULL;
    if (address(w[i].tiles) % 16 || address(w[i].scales) % 4 || address(w[i].zeros) % 2) return SWIGLU_B200_ERR_ALIGN;
  }
  return SWIGLU_B200_OK;
}

// Ranges that a call reads of one matrix.
int weight_ranges(const W4& w, const W4Shape& s, ByteRange* r) {
  const long long tiles = (s.n + kTileRows - 1) / kTileRows * s.col_tiles;
  const long long groups = (tiles << s.groups_log2) * kTileRows;
  r[0] = byte_range(w.tiles, 1, tiles * kTileBytes, 0);
  r[1] = byte_range(w.scales, 1, groups * 2, 0);
  r[2] = w.zeros ? byte_range(w.zeros, 1, groups, 0) : ByteRange{0, 0};
  return 3;
}

template <class T, int MATS, int NT, int ACT>
int launch(void* y, const void* x, const W4* w, const W4Shape& s, float gm, float dm, cudaStream_t st) {
  // Two weight tiles to a warp where a token tile of 32 is read beside them: its fragments are 8 KB per column tile, 8
  // times the weights of one tile.
  constexpr int RT = NT == 4 && MATS == 1 ? 2 : 1;
  const long long row_tiles = (s.n + kTileRows - 1) / kTileRows;
  const long long gx = (row_tiles + RT - 1) / RT, gy = (s.m + 8 * NT - 1) / (8 * NT);
  if (gx > 0x7fffffffLL || gy > 65535) return SWIGLU_B200_ERR_SHAPE;
  w4_kernel<T, MATS, RT, NT, ACT><<<dim3((unsigned)gx, (unsigned)gy), 32 * kWarps, 0, st>>>(
      y, x, w[0], MATS == 2 ? w[1] : w[0], s, gm, dm);
  return launched();
}

template <int MATS, int ACT>
int run(void* y, const void* x, const W4* w, W4Shape s, int64_t m, int64_t x_row_stride, int64_t y_row_stride,
        int dtype, float gm, float dm, int device, void* stream) {
  if (m < 0) return SWIGLU_B200_ERR_SHAPE;
  if (m == 0 || s.n == 0) return SWIGLU_B200_OK;
  if (s.k == 0) return SWIGLU_B200_ERR_SHAPE;
  if (x_row_stride < s.k || y_row_stride < s.n) return SWIGLU_B200_ERR_SHAPE;
  if (!fits_address_space(m, x_row_stride, 2) || !fits_address_space(m, y_row_stride, 2)) return SWIGLU_B200_ERR_SHAPE;
  if (!y || !x) return SWIGLU_B200_ERR_NULL;
  if (address(y) % 2 || address(x) % 2) return SWIGLU_B200_ERR_ALIGN;
  const ByteRange out = byte_range(y, m, s.n * 2, y_row_stride * 2);
  ByteRange in[7];
  in[0] = byte_range(x, m, s.k * 2, x_row_stride * 2);
  int count = 1;
  for (int i = 0; i < MATS; ++i) count += weight_ranges(w[i], s, in + count);
  for (int i = 0; i < count; ++i)
    if (overlap(out, in[i])) return SWIGLU_B200_ERR_ALIAS;
  CallDevice scope(device);
  if (scope.err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_DEVICE, scope.err);
  s.m = m;
  s.x_pitch = x_row_stride;
  s.y_pitch = y_row_stride;
  s.x_vec = address(x) % 16 == 0 && (m == 1 || x_row_stride % 8 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto typed = [&](auto t) {
    using T = decltype(t);
    if (m <= 8) return launch<T, MATS, 1, ACT>(y, x, w, s, gm, dm, st);
    if (m <= 16) return launch<T, MATS, 2, ACT>(y, x, w, s, gm, dm, st);
    return launch<T, MATS, 4, ACT>(y, x, w, s, gm, dm, st);
  };
  return dtype == SWIGLU_B200_F16 ? typed(__half{}) : typed(__nv_bfloat16{});
}

}  // namespace

extern "C" {

int swiglu_b200_w4_linear(void* y, const void* x, const void* tiles, const void* scales, const void* zeros, int64_t m,
                          int64_t n, int64_t k, int64_t x_row_stride, int64_t y_row_stride, int group, int dtype,
                          int device, void* stream) {
  const W4 w{tiles, scales, zeros};
  W4Shape s{};
  const int rc = check(&w, 1, n, k, group, dtype, s);
  if (rc != SWIGLU_B200_OK) return rc;
  return run<1, ACT_SILU>(y, x, &w, s, m, x_row_stride, y_row_stride, dtype, 1.0f, 1.0f, device, stream);
}

int swiglu_b200_w4_gate_up(void* h, const void* x, const void* gate_tiles, const void* gate_scales,
                           const void* gate_zeros, const void* up_tiles, const void* up_scales, const void* up_zeros,
                           int64_t m, int64_t n, int64_t k, int64_t x_row_stride, int64_t h_row_stride, int group,
                           int dtype, int activation, float gm, float dm, int device, void* stream) {
  const W4 w[2] = {{gate_tiles, gate_scales, gate_zeros}, {up_tiles, up_scales, up_zeros}};
  W4Shape s{};
  const int rc = check(w, 2, n, k, group, dtype, s);
  if (rc != SWIGLU_B200_OK) return rc;
  switch (activation) {
    case SWIGLU_B200_SILU:
      return run<2, ACT_SILU>(h, x, w, s, m, x_row_stride, h_row_stride, dtype, gm, dm, device, stream);
    case SWIGLU_B200_GELU_TANH:
      return run<2, ACT_GELU_TANH>(h, x, w, s, m, x_row_stride, h_row_stride, dtype, gm, dm, device, stream);
    case SWIGLU_B200_GELU_ERF:
      return run<2, ACT_GELU_ERF>(h, x, w, s, m, x_row_stride, h_row_stride, dtype, gm, dm, device, stream);
    default: return SWIGLU_B200_ERR_ARG;
  }
}

int swiglu_b200_w4_dequantize(void* out, const void* tiles, const void* scales, const void* zeros, int64_t n,
                              int64_t k, int64_t out_row_stride, int group, int dtype, int device, void* stream) {
  const W4 w{tiles, scales, zeros};
  W4Shape s{};
  const int rc = check(&w, 1, n, k, group, dtype, s);
  if (rc != SWIGLU_B200_OK) return rc;
  if (n == 0 || k == 0) return SWIGLU_B200_OK;
  if (out_row_stride < k || !fits_address_space(n, out_row_stride, 2)) return SWIGLU_B200_ERR_SHAPE;
  if (!out) return SWIGLU_B200_ERR_NULL;
  if (address(out) % 2) return SWIGLU_B200_ERR_ALIGN;
  const ByteRange o = byte_range(out, n, k * 2, out_row_stride * 2);
  ByteRange in[3];
  weight_ranges(w, s, in);
  for (const ByteRange& r : in)
    if (overlap(o, r)) return SWIGLU_B200_ERR_ALIAS;
  const long long tiles_all = (n + kTileRows - 1) / kTileRows * s.col_tiles, ctas = (tiles_all + 7) / 8;
  if (ctas > 0x7fffffffLL) return SWIGLU_B200_ERR_SHAPE;
  CallDevice scope(device);
  if (scope.err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_DEVICE, scope.err);
  s.y_pitch = out_row_stride;
  const int vec = address(out) % 16 == 0 && out_row_stride % 8 == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == SWIGLU_B200_F16) w4_dequantize_kernel<__half><<<(unsigned)ctas, 256, 0, st>>>(out, w, s, vec);
  else w4_dequantize_kernel<__nv_bfloat16><<<(unsigned)ctas, 256, 0, st>>>(out, w, s, vec);
  return launched();
}

}  // extern "C"
