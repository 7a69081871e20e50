// Gated activations whose inputs are kept in 8 bits between the passes (declarations: include/swiglu_b200.h).
//
// The forward reads gate and up, writes h = act(gate*gm) * up * dm from the values as they came, and beside it an
// 8-bit copy of both inputs; the backward reads that copy in the inputs' place.  Per row, 32 consecutive columns
// (a group; the last one of a row may be short) share one step:
//   a     = largest magnitude of the group
//   E     = biased fp32 exponent of a, plus one where a would round to 128 steps, minus 6, at least 1
//   code  = rint(x * 2^(127-E)), in [-127, 127]                 value = code * 2^(E-127)
// so the error is at most half a step, a/127 at worst.  The step is a power of two on purpose: scaling by it is
// exact, so the only rounding is rint and every implementation of these two lines gives the same codes.  Codes are
// int8, E is one byte per group; 8.25 bits per element instead of 16 or 32.  A group that holds an Inf, a NaN or a
// magnitude that would round to 2^128 (E above 248) stores E = 255 and reads back as NaN, so the gradients of a step
// that overflowed do not come out finite.
//
// The kernels are pure streams.  Bytes per element of size s: forward 2s read + s + 2*33/32 written (8.06 for bf16),
// backward s + 2*33/32 read + 2s written (8.06), with h recomputed one s more.  A lane owns one 32-byte frame of each
// full-width tensor (16 columns in 16 bits, 8 in fp32), so a group is 2 or 4 neighbouring lanes and its maximum takes
// one or two shuffles; the lane's codes are one 16- or 8-byte access.  Where every row of every tensor starts on a
// 32-byte boundary frames are loaded and stored as they are (and contiguous rows of whole groups are one long row);
// otherwise (SKEW) they are read through the 48-byte windows and written through the realigned stores of
// swiglu_kernels.cuh, with the last partial frame of a row moved element by element by one lane.
#include "swiglu_b200.h"

#include <type_traits>

#include "launch_common.cuh"
#include "swiglu_kernels.cuh"

namespace {

using namespace swiglu_b200;

constexpr int kGroup = 32;     // columns that share a step
constexpr uint32_t kMaxExponent = 248;  // 127 steps of 2^(248-127) are below 2^128, 64 steps of the next are not
constexpr uint32_t kNonFinite = 255;

struct Ckpt8Shape {
  long long rows, cols;
  long long groups;      // per row; a row of codes takes 32 * groups bytes, a row of step exponents `groups`
  long long pitch_in;    // bytes between rows of gate / up (forward) or dh (backward)
  long long pitch_out;   // bytes between rows of h
  long long pitch_grad;  // bytes between rows of dgate / dup
};

// Largest magnitude among the lane's elements as the bit pattern of a float; NaN and Inf order above every finite
// value.
template <class T> __device__ __forceinline__ uint32_t top_bits(const Vec<32>& v);
template <> __device__ __forceinline__ uint32_t top_bits<float>(const Vec<32>& v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, v.w[i] & 0x7fffffffu);
  return m;
}
template <> __device__ __forceinline__ uint32_t top_bits<__nv_bfloat16>(const Vec<32>& v) {
  __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v.w[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&v.w[i])));
  const uint32_t w = *reinterpret_cast<uint32_t*>(&m);
  return max(w << 16, w & 0xffff0000u) & 0x7fffffffu;
}
template <> __device__ __forceinline__ uint32_t top_bits<__half>(const Vec<32>& v) {
  __half2 m = __habs2(*reinterpret_cast<const __half2*>(&v.w[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&v.w[i])));
  const float2 f = __half22float2(m);
  return max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu);
}

// The group's E from its largest magnitude.  0x10000 is half a step of 127 at that exponent: added to the bit pattern
// it carries into the exponent exactly when the magnitude would round to 128 steps.
__device__ __forceinline__ uint32_t step_exponent(uint32_t top) {
  const int e = (int)((top + 0x10000u) >> 23) - 6;
  return e > (int)kMaxExponent ? kNonFinite : (uint32_t)max(e, 1);
}

// Codes of EPV floats, four to a word.  x * 2^(127-E) is exact; adding 1.5 * 2^23 rounds it to an integer (to
// nearest, ties to even) and leaves that integer's two's complement in the low byte.
template <int EPV>
__device__ __forceinline__ void encode(const float* f, uint32_t e, uint32_t* codes) {
  const float inv = __uint_as_float((254u - min(e, 254u)) << 23);  // 0 for a non-finite group: its codes do not matter
#pragma unroll
  for (int i = 0; i < EPV / 4; ++i) {
    uint32_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = __float_as_uint(fmaf(f[4 * i + j], inv, 12582912.0f));
    codes[i] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
  }
}

// Values of 4 * WORDS codes.  code + 128 as the low byte of 2^23 is a float whose difference to 2^23 + 128 is the code;
// times the step both operations are exact (folding them into one FMA would overflow for steps above 2^104).
template <int WORDS>
__device__ __forceinline__ void decode(const uint32_t* codes, uint32_t e, float* f) {
  const float step = __uint_as_float(e == kNonFinite ? 0x7fffffffu : e << 23);
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    const uint32_t w = codes[i] ^ 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      f[4 * i + j] = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 | j)) - 8388736.0f) * step;
  }
}

// Position of a lane: its row, its frame in the row, and how much of the row that frame covers.
template <class T>
struct Place {
  static constexpr int EPV = 32 / (int)sizeof(T);
  long long row, v;
  bool in_row;   // the frame's group exists (its codes are stored, zeros past the last column)
  bool full;     // all EPV columns exist
  int rest;      // columns of a partial frame, 0 for any other
  bool first, last;  // no full frame of the same task before / after this one
  bool whole;        // every lane of the task has a full frame (uniform over the warp)
  __device__ __forceinline__ explicit Place(const Ckpt8Shape& s) {
    const int lane = threadIdx.x & 31;
    const int task = (int)blockIdx.x * (int)(blockDim.x >> 5) + (int)(threadIdx.x >> 5);
    row = (long long)blockIdx.y + (long long)blockIdx.z * gridDim.y;
    v = (long long)task * 32 + lane;
    const long long n_full = s.cols / EPV;
    in_row = v < s.groups * (kGroup / EPV);
    full = v < n_full;
    rest = v == n_full ? (int)(s.cols % EPV) : 0;
    first = lane == 0;
    last = lane == 31 || v == n_full - 1;
    whole = (long long)task * 32 + 32 <= n_full;
  }
};

// The lane's frame of a row that starts at `row`; columns that do not exist read as zero.  In a WHOLE task every lane
// has a full frame, which it reads as the two or three aligned 16-byte pieces it lies in.
struct Pieces {
  Vec<16> p[3];
};
template <class T, bool SKEW, bool WHOLE> struct Frame {
  Window w;
  Pieces q;

  template <int LDM> __device__ __forceinline__ void issue(const char* row, const Place<T>& at) {
    if constexpr (WHOLE && !SKEW) {
      w.main = Ld<32, LDM>::ld(row + at.v * 32);
    } else if constexpr (WHOLE) {
      const char* p = row + at.v * 32 - ((uintptr_t)row & 15);
      q.p[0] = Ld<16, LDM>::ld(p);
      q.p[1] = Ld<16, LDM>::ld(p + 16);
      q.p[2] = ((uintptr_t)row & 15) ? Ld<16, LDM>::ld(p + 32) : q.p[1];
    } else if constexpr (!SKEW) {
      if (at.full) w.main = Ld<32, LDM>::ld(row + at.v * 32);
      else w.main = Vec<32>{};
    } else {
      w.main = Vec<32>{};
      w.nb = Vec<16>{};
      ld_window_issue<LDM>(row, at.v, (int)((uintptr_t)row & 31), at.full, w);
    }
  }
  __device__ __forceinline__ Vec<32> finish(const char* row, const Place<T>& at) const {
    if constexpr (!SKEW) {
      return w.main;
    } else if constexpr (WHOLE) {
      const uint32_t x[12] = {q.p[0].w[0], q.p[0].w[1], q.p[0].w[2], q.p[0].w[3], q.p[1].w[0], q.p[1].w[1],
                              q.p[1].w[2], q.p[1].w[3], q.p[2].w[0], q.p[2].w[1], q.p[2].w[2], q.p[2].w[3]};
      return shift_window(x, (int)((uintptr_t)row & 15));
    } else {
      constexpr int ES = (int)sizeof(T);
      Vec<32> v = ld_window_finish(w, (int)((uintptr_t)row & 31));  // zero where nothing was loaded
      if (at.rest) {
        const char* p = row + at.v * 32;
#pragma unroll
        for (int e = 0; e < Place<T>::EPV; ++e)
          if (e < at.rest) {
            const uint32_t x = Ld<ES, LD_PLAIN>::ld(p + e * ES).w[0];
            v.w[e * ES / 4] |= (e * ES % 4) ? x << 16 : x;
          }
      }
      return v;
    }
  }
};

// Stores the lane's frame into a row that starts at `row`.  All 32 lanes call this together.
template <class T, bool SKEW, bool WHOLE>
__device__ __forceinline__ void frame_store(char* row, const Place<T>& at, const Vec<32>& v) {
  if constexpr (!SKEW) {
    if (WHOLE || at.full) St<32, ST_CS>::st(row + at.v * 32, v);
  } else {
    constexpr int ES = (int)sizeof(T);
    char* p = row + at.v * 32;
    if constexpr (WHOLE) {
      const int lane = threadIdx.x & 31;
      st_skewed32<ST_CS>(p, v, (int)((uintptr_t)row & 31), true, lane == 0, lane == 31);
    } else {
      st_skewed32<ST_CS>(p, v, (int)((uintptr_t)row & 31), at.full, at.first, at.last);
      if (at.rest) {
#pragma unroll
        for (int e = 0; e < Place<T>::EPV; ++e)
          if (e < at.rest) {
            Vec<ES> x;
            x.w[0] = (e * ES % 4) ? v.w[e * ES / 4] >> 16 : v.w[e * ES / 4];
            if constexpr (ES == 2) x.w[0] &= 0xffffu;
            St<ES, ST_PLAIN>::st(p + e * ES, x);
          }
      }
    }
  }
}

// E of the group this lane belongs to.  All 32 lanes call this together; a group never crosses a warp.
template <class T>
__device__ __forceinline__ uint32_t group_exponent(const Vec<32>& v) {
  uint32_t top = top_bits<T>(v);
#pragma unroll
  for (int d = 1; d < kGroup / Place<T>::EPV; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  return step_exponent(top);
}

template <class T, bool WHOLE>
__device__ __forceinline__ void codes_store(void* codes, void* steps, const Ckpt8Shape& s, const Place<T>& at,
                                            const float* f, uint32_t e) {
  constexpr int EPV = Place<T>::EPV;
  if (!WHOLE && !at.in_row) return;
  Vec<EPV> c;
  encode<EPV>(f, e, c.w);
  St<EPV, ST_CS>::st(byte(codes) + at.row * s.groups * kGroup + at.v * EPV, c);
  if (at.v % (kGroup / EPV) == 0) {
    Vec<2> b;
    b.w[0] = e;
    asm volatile("st.global.u8 [%0], %1;" ::"l"(byte(steps) + at.row * s.groups + at.v / (kGroup / EPV)), "r"(b.w[0])
                 : "memory");
  }
}

template <class T, bool WHOLE>
__device__ __forceinline__ uint32_t step_load(const void* steps, const Ckpt8Shape& s, const Place<T>& at) {
  uint32_t e = 1;
  if (WHOLE || at.in_row)
    asm volatile("ld.global.nc.u8 %0, [%1];"
                 : "=r"(e) : "l"(cbyte(steps) + at.row * s.groups + at.v / (kGroup / Place<T>::EPV)));
  return e;
}

constexpr int kWarps = 4;  // most warps of a CTA

// CTAs to an SM that the registers are budgeted for.  bf16 [16384, 14336], 6 / 8 / 10 / 16 of them: forward 283 / 276 / 277 /
// 304 us; backward with 6 / 8 / 10 / 12: 385 / 301 / 289 / 292 us, and at half-width 11009 packed 103 / 90 / 77 / 78 us.
constexpr int kCtas = 10;

template <class T, int ACT, bool SKEW, bool WHOLE>
__device__ __forceinline__ void forward_task(void* h, void* gate_codes, void* up_codes, void* gate_steps, void* up_steps,
                                             const void* gate, const void* up, const Ckpt8Shape& s, const Place<T>& at,
                                             float gm, float dm) {
  constexpr bool FAST = (sizeof(T) == 2);
  constexpr int EPV = Place<T>::EPV;
  const Consts c(gm, dm);
  const char* gate_row = cbyte(gate) + at.row * s.pitch_in;
  const char* up_row = cbyte(up) + at.row * s.pitch_in;
  Frame<T, SKEW, WHOLE> wg, wu;
  wg.template issue<LD_PLAIN>(gate_row, at);
  wu.template issue<LD_PLAIN>(up_row, at);
  const Vec<32> vg = wg.finish(gate_row, at), vu = wu.finish(up_row, at);
  const uint32_t eg = group_exponent<T>(vg), eu = group_exponent<T>(vu);
  float fg[EPV], fu[EPV];
  Codec<T>::template unpack<32>(vg, fg);
  Codec<T>::template unpack<32>(vu, fu);
  codes_store<T, WHOLE>(gate_codes, gate_steps, s, at, fg, eg);
  codes_store<T, WHOLE>(up_codes, up_steps, s, at, fu, eu);
  if (h != nullptr) {
    float fh[EPV];
#pragma unroll
    for (int i = 0; i < EPV; ++i) fh[i] = Math<FAST, ACT>::fwd(fg[i], fu[i], c);
    Vec<32> vh;
    Codec<T>::template pack<32>(fh, vh);
    frame_store<T, SKEW, WHOLE>(byte(h) + at.row * s.pitch_out, at, vh);
  }
}

// h may be NULL: the codes alone are stored.  Tasks without a row's end take a copy of the code that has no predicates.
template <class T, int ACT, bool SKEW>
__global__ void __launch_bounds__(32 * kWarps, kCtas)
ckpt8_fwd_kernel(void* h, void* gate_codes, void* up_codes, void* gate_steps, void* up_steps,
                 const void* __restrict__ gate, const void* __restrict__ up, Ckpt8Shape s, float gm, float dm) {
  const Place<T> at(s);
  if (at.row >= s.rows) return;
  if (at.whole) forward_task<T, ACT, SKEW, true>(h, gate_codes, up_codes, gate_steps, up_steps, gate, up, s, at, gm, dm);
  else forward_task<T, ACT, SKEW, false>(h, gate_codes, up_codes, gate_steps, up_steps, gate, up, s, at, gm, dm);
}

template <class T, int ACT, bool SKEW, bool H, bool WHOLE>
__device__ __forceinline__ void backward_task(void* h, void* dgate, void* dup, const void* dout, const void* gate_codes,
                                              const void* up_codes, const void* gate_steps, const void* up_steps,
                                              const Ckpt8Shape& s, const Place<T>& at, float gm, float dm) {
  constexpr bool FAST = (sizeof(T) == 2);
  constexpr int EPV = Place<T>::EPV;
  const Consts c(gm, dm);
  const char* dout_row = cbyte(dout) + at.row * s.pitch_in;
  Frame<T, SKEW, WHOLE> wd;
  wd.template issue<LD_PLAIN>(dout_row, at);
  Vec<EPV> cg{}, cu{};
  if (WHOLE || at.in_row) {
    const long long off = at.row * s.groups * kGroup + at.v * EPV;
    cg = Ld<EPV, LD_NC_NOALLOC>::ld(cbyte(gate_codes) + off);
    cu = Ld<EPV, LD_NC_NOALLOC>::ld(cbyte(up_codes) + off);
  }
  const uint32_t eg = step_load<T, WHOLE>(gate_steps, s, at), eu = step_load<T, WHOLE>(up_steps, s, at);
  const Vec<32> vd = wd.finish(dout_row, at);
  float fg[EPV], fu[EPV], fd[EPV], fdg[EPV], fdu[EPV], fh[EPV];
  decode<EPV / 4>(cg.w, eg, fg);
  decode<EPV / 4>(cu.w, eu, fu);
  Codec<T>::template unpack<32>(vd, fd);
#pragma unroll
  for (int i = 0; i < EPV; ++i) {
    if constexpr (H) Math<FAST, ACT>::bwd_h(fd[i], fg[i], fu[i], c, fh[i], fdg[i], fdu[i]);
    else Math<FAST, ACT>::bwd(fd[i], fg[i], fu[i], c, fdg[i], fdu[i]);
  }
  Vec<32> x;
  Codec<T>::template pack<32>(fdg, x);
  frame_store<T, SKEW, WHOLE>(byte(dgate) + at.row * s.pitch_grad, at, x);
  Codec<T>::template pack<32>(fdu, x);
  frame_store<T, SKEW, WHOLE>(byte(dup) + at.row * s.pitch_grad, at, x);
  if constexpr (H) {
    Codec<T>::template pack<32>(fh, x);
    frame_store<T, SKEW, WHOLE>(byte(h) + at.row * s.pitch_out, at, x);
  }
}

// With H, h = act(gate*gm) * up * dm of the kept values is stored too; it may overwrite dout (a warp stores only
// elements whose values its own lanes have read by then).  The copy of the code for whole tasks pays for aligned rows
// (289 -> 276 us); the skewed form is issue-bound and twice its size overflows the instruction cache (with h, half-width
// 11009 packed: 105 -> 133 us), so it has one copy.
template <class T, int ACT, bool SKEW, bool H>
__global__ void __launch_bounds__(32 * kWarps, kCtas)
ckpt8_bwd_kernel(void* h, void* dgate, void* dup, const void* dout, const void* __restrict__ gate_codes,
                 const void* __restrict__ up_codes, const void* __restrict__ gate_steps,
                 const void* __restrict__ up_steps, Ckpt8Shape s, float gm, float dm) {
  const Place<T> at(s);
  if (at.row >= s.rows) return;
  if (!SKEW && at.whole)
    backward_task<T, ACT, SKEW, H, !SKEW>(h, dgate, dup, dout, gate_codes, up_codes, gate_steps, up_steps, s, at, gm, dm);
  else
    backward_task<T, ACT, SKEW, H, false>(h, dgate, dup, dout, gate_codes, up_codes, gate_steps, up_steps, s, at, gm, dm);
}

// ------------------------------------------------------------------ host side

struct Grid {
  dim3 grid;
  unsigned block;
  bool ok;  // within the limits of a launch
};

// A CTA takes up to kWarps consecutive tasks of one row, the row's tasks spread evenly over its CTAs.
Grid grid_of(const Ckpt8Shape& s, int epv) {
  const long long frames = s.groups * (kGroup / epv);
  const long long tasks = (frames + 31) / 32;
  const long long ctas = (tasks + kWarps - 1) / kWarps;
  const long long warps = (tasks + ctas - 1) / ctas;
  const long long z = (s.rows + 65534) / 65535;
  const long long y = (s.rows + z - 1) / z;
  return Grid{dim3((unsigned)ctas, (unsigned)y, (unsigned)z), (unsigned)(32 * warps),
              tasks <= 0x7fffffffLL && z <= 65535};
}

bool known_dtype(int dtype) {
  return dtype == SWIGLU_B200_F32 || dtype == SWIGLU_B200_F16 || dtype == SWIGLU_B200_BF16;
}

template <class F>
int by_activation(int activation, F&& f) {
  switch (activation) {
    case ACT_SILU: return f(std::integral_constant<int, ACT_SILU>{});
    case ACT_GELU_TANH: return f(std::integral_constant<int, ACT_GELU_TANH>{});
    default: return f(std::integral_constant<int, ACT_GELU_ERF>{});
  }
}
template <class F>
int by_dtype(int dtype, F&& f) {
  switch (dtype) {
    case SWIGLU_B200_F32: return f(float{});
    case SWIGLU_B200_F16: return f(__half{});
    default: return f(__nv_bfloat16{});
  }
}

// True when rows can be taken as one: contiguous everywhere and made of whole groups.
bool one_row(long long rows, long long cols, const long long* pitch, int n) {
  if (cols % kGroup) return false;
  for (int i = 0; i < n; ++i)
    if (rows > 1 && pitch[i] != cols) return false;
  return true;
}

}  // namespace

extern "C" {

int swiglu_b200_ckpt8_fwd(void* h, void* gate_codes, void* up_codes, void* gate_steps, void* up_steps,
                          const void* gate, const void* up, int64_t rows, int64_t cols, int64_t in_row_stride,
                          int64_t out_row_stride, int dtype, int activation, float gm, float dm, int device,
                          void* stream) {
  if (!known_dtype(dtype)) return SWIGLU_B200_ERR_DTYPE;
  if (activation < SWIGLU_B200_SILU || activation > SWIGLU_B200_GELU_ERF) return SWIGLU_B200_ERR_ARG;
  if (rows < 0 || cols < 0) return SWIGLU_B200_ERR_SHAPE;
  if (rows == 0 || cols == 0) return SWIGLU_B200_OK;
  if (in_row_stride < cols || (h && out_row_stride < cols)) return SWIGLU_B200_ERR_SHAPE;
  const int es = dtype == SWIGLU_B200_F32 ? 4 : 2;
  if (!fits_address_space(rows, in_row_stride, es) || (h && !fits_address_space(rows, out_row_stride, es)))
    return SWIGLU_B200_ERR_SHAPE;
  if (!gate_codes || !up_codes || !gate_steps || !up_steps || !gate || !up) return SWIGLU_B200_ERR_NULL;
  if (address(gate) % es || address(up) % es || address(h) % es || address(gate_codes) % 16 ||
      address(up_codes) % 16)
    return SWIGLU_B200_ERR_ALIGN;
  const long long groups = (cols + kGroup - 1) / kGroup;
  {
    const ByteRange in[2] = {byte_range(gate, rows, cols * es, in_row_stride * es),
                             byte_range(up, rows, cols * es, in_row_stride * es)};
    ByteRange out[5] = {byte_range(gate_codes, 1, rows * groups * kGroup, 0),
                        byte_range(up_codes, 1, rows * groups * kGroup, 0),
                        byte_range(gate_steps, 1, rows * groups, 0), byte_range(up_steps, 1, rows * groups, 0),
                        h ? byte_range(h, rows, cols * es, out_row_stride * es) : ByteRange{0, 0}};
    for (int i = 0; i < 5; ++i) {
      if (overlap(out[i], in[0]) || overlap(out[i], in[1])) return SWIGLU_B200_ERR_ALIAS;
      for (int j = 0; j < i; ++j)
        if (overlap(out[i], out[j])) return SWIGLU_B200_ERR_ALIAS;
    }
  }
  CallDevice scope(device);
  if (scope.err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_DEVICE, scope.err);

  Ckpt8Shape s{};
  const long long pitches[2] = {in_row_stride, h ? out_row_stride : cols};
  const bool flat = one_row(rows, cols, pitches, 2);
  s.rows = flat ? 1 : rows;
  s.cols = flat ? rows * cols : cols;
  s.groups = flat ? rows * groups : groups;
  s.pitch_in = in_row_stride * es;
  s.pitch_out = pitches[1] * es;
  const bool pitched = s.rows > 1;
  const bool skew = address(gate) % 32 || address(up) % 32 || address(h) % 32 || (cols * es) % 32 ||
                    (pitched && (s.pitch_in % 32 || s.pitch_out % 32));
  const Grid g = grid_of(s, 32 / es);
  if (!g.ok) return SWIGLU_B200_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_activation(activation, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      if (skew)
        ckpt8_fwd_kernel<T, ACT, true><<<g.grid, g.block, 0, st>>>(h, gate_codes, up_codes, gate_steps, up_steps, gate, up, s, gm, dm);
      else
        ckpt8_fwd_kernel<T, ACT, false><<<g.grid, g.block, 0, st>>>(h, gate_codes, up_codes, gate_steps, up_steps, gate, up, s, gm, dm);
      return launched();
    });
  });
}

int swiglu_b200_ckpt8_bwd(void* h, void* dgate, void* dup, const void* dout, const void* gate_codes,
                          const void* up_codes, const void* gate_steps, const void* up_steps, int64_t rows,
                          int64_t cols, int64_t grad_row_stride, int64_t dout_row_stride, int64_t h_row_stride,
                          int dtype, int activation, float gm, float dm, int device, void* stream) {
  if (!known_dtype(dtype)) return SWIGLU_B200_ERR_DTYPE;
  if (activation < SWIGLU_B200_SILU || activation > SWIGLU_B200_GELU_ERF) return SWIGLU_B200_ERR_ARG;
  if (rows < 0 || cols < 0) return SWIGLU_B200_ERR_SHAPE;
  if (rows == 0 || cols == 0) return SWIGLU_B200_OK;
  if (grad_row_stride < cols || dout_row_stride < cols || (h && h_row_stride < cols)) return SWIGLU_B200_ERR_SHAPE;
  const int es = dtype == SWIGLU_B200_F32 ? 4 : 2;
  if (!fits_address_space(rows, grad_row_stride, es) || !fits_address_space(rows, dout_row_stride, es) ||
      (h && !fits_address_space(rows, h_row_stride, es)))
    return SWIGLU_B200_ERR_SHAPE;
  if (!dgate || !dup || !dout || !gate_codes || !up_codes || !gate_steps || !up_steps) return SWIGLU_B200_ERR_NULL;
  if (address(dgate) % es || address(dup) % es || address(dout) % es || address(h) % es ||
      address(gate_codes) % 16 || address(up_codes) % 16)
    return SWIGLU_B200_ERR_ALIGN;
  const long long groups = (cols + kGroup - 1) / kGroup;
  {
    const ByteRange d = byte_range(dout, rows, cols * es, dout_row_stride * es);
    const ByteRange in[4] = {byte_range(gate_codes, 1, rows * groups * kGroup, 0),
                             byte_range(up_codes, 1, rows * groups * kGroup, 0),
                             byte_range(gate_steps, 1, rows * groups, 0), byte_range(up_steps, 1, rows * groups, 0)};
    // rows of a packed dgate|dup buffer lie between one another's: as ranges the two overlap rightly
    const ByteRange grad[2] = {byte_range(dgate, rows, cols * es, grad_row_stride * es),
                               byte_range(dup, rows, cols * es, grad_row_stride * es)};
    if (rows_overlap(dgate, dup, rows, cols * es, grad_row_stride * es)) return SWIGLU_B200_ERR_ALIAS;
    const ByteRange hr = h ? byte_range(h, rows, cols * es, h_row_stride * es) : ByteRange{0, 0};
    const bool over_dout = h == dout && h_row_stride == dout_row_stride;
    for (const ByteRange& g : grad)
      if (overlap(g, d) || overlap(g, hr)) return SWIGLU_B200_ERR_ALIAS;
    if (h && !over_dout && overlap(hr, d)) return SWIGLU_B200_ERR_ALIAS;
    for (const ByteRange& r : in)
      if (overlap(r, grad[0]) || overlap(r, grad[1]) || overlap(r, hr)) return SWIGLU_B200_ERR_ALIAS;
  }
  CallDevice scope(device);
  if (scope.err != cudaSuccess) return note_cuda_error(SWIGLU_B200_ERR_DEVICE, scope.err);

  Ckpt8Shape s{};
  const long long pitches[3] = {grad_row_stride, dout_row_stride, h ? h_row_stride : cols};
  const bool flat = one_row(rows, cols, pitches, 3);
  s.rows = flat ? 1 : rows;
  s.cols = flat ? rows * cols : cols;
  s.groups = flat ? rows * groups : groups;
  s.pitch_in = dout_row_stride * es;
  s.pitch_out = pitches[2] * es;
  s.pitch_grad = grad_row_stride * es;
  const bool pitched = s.rows > 1;
  const bool skew = address(dgate) % 32 || address(dup) % 32 || address(dout) % 32 || address(h) % 32 ||
                    (cols * es) % 32 ||
                    (pitched && (s.pitch_in % 32 || s.pitch_out % 32 || s.pitch_grad % 32));
  const Grid g = grid_of(s, 32 / es);
  if (!g.ok) return SWIGLU_B200_ERR_SHAPE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return by_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return by_activation(activation, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      auto launch = [&](auto kernel) {
        kernel<<<g.grid, g.block, 0, st>>>(h, dgate, dup, dout, gate_codes, up_codes, gate_steps, up_steps, s, gm, dm);
      };
      if (h) skew ? launch(ckpt8_bwd_kernel<T, ACT, true, true>) : launch(ckpt8_bwd_kernel<T, ACT, false, true>);
      else skew ? launch(ckpt8_bwd_kernel<T, ACT, true, false>) : launch(ckpt8_bwd_kernel<T, ACT, false, false>);
      return launched();
    });
  });
}

}  // extern "C"
