// dc_adamw.hip — one AdamW step over many tensors at once, states in 32 bits or in 8 bits with scales.
//
// Memory-bound: an element with 32-bit states moves 28 bytes (gradient 2; param, m, v in and out 24; the bf16 copy 2),
// with 8-bit ones 16. The tensors' addresses travel in the kernel's arguments, kTensors a launch, so a step of a whole
// model is a few launches, nothing is uploaded and nothing is kept between calls. A workgroup takes kChunk elements of one
// tensor (found from the tensors' first chunks); a wave's 64 lanes take 4 neighbouring
// elements each, which is one 8-bit state block: its maximum is a DPP reduction, and a state's codes and scale are read
// and written once. What the next step alone reads again passes the caches by (non-temporal); the bf16 copy does not.
//
// Measured, us (TB/s of the 28 and 16.06 bytes an element): 134M elements, 32-bit states 647 (5.8), 8-bit 368 (5.9); 484 thousand in
// 30 tensors 4.5 and 4.8, which is the launch's. A block a wave; four blocks a wave, all loaded first: 699, 374, 7.1, 9.2;
// that through the caches 718, 401.
#include <algorithm>
#include <cmath>

#include "dc_internal.hpp"
#include "dc_numeric.hpp"

namespace {

using dc::bf16;

constexpr int kTensors = 48;  // of a launch: their table, 3.5 KiB, travels in the kernel's arguments
constexpr int kThreads = 256;
constexpr int kBlock = DC_ADAMW_BLOCK;
constexpr int kChunk = kThreads / 64 * kBlock;
static_assert(kBlock == 64 * 4, "a wave's lanes take four elements each of a block");

struct Tensor {
  float* param;
  const void* grad;
  void *m, *v;
  float *m_scales, *v_scales;
  uint16_t* copy;
  int64_t n;
  int64_t grad_f32;
};

struct Step {
  float beta1, beta2, rest1, rest2;  // rest: 1 - beta
  float rate, root, eps, decay;      // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), eps, 1 - lr weight_decay
  float grad_scale;
  int32_t count;
  uint32_t first[kTensors];  // chunk of each tensor in the launch
  Tensor t[kTensors];
};

// Four 8-bit states with their scale.
__device__ inline void unpack_fp8(uint32_t w, float (&v)[4]) {
  const dc::f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
}

// A block's scale is its largest magnitude times 1 / 448, and its values are held as their products with 448 times the reciprocal
// of that magnitude (at most the largest float, where the scale is 2^-128, and zeros stay zeros): products, where the definition
// divides, are within an ulp of it, far below a code's step.
__device__ inline float state_scale(float top) {
  const float s = top * (1.0f / dc::kFp8Top);
  return top > 0.0f && s < 0x1p-128f ? 0x1p-128f : s;
}
__device__ inline float state_factor(float top) {
  const float f = (1.0f / top) * dc::kFp8Top;
  return f > __FLT_MAX__ ? __FLT_MAX__ : f;
}

// The elements [0, 4) at p of which `left` exist; zeros for the others.
template <typename T>
__device__ inline void load4(const T* p, int64_t left, float (&v)[4]);
template <>
__device__ inline void load4(const float* p, int64_t left, float (&v)[4]) {
  if (left >= 4) {
    const dc::f32x4_at4 w = __builtin_nontemporal_load(reinterpret_cast<const dc::f32x4_at4*>(p));
    v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
  } else {
    dc::load_some(p, left, v);
  }
}
__device__ inline void store4(float* p, int64_t left, const float (&v)[4]) {
  if (left >= 4) {
    const dc::f32x4 w = {v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(w, reinterpret_cast<dc::f32x4_at4*>(p));
  } else {
    dc::store_some(p, left, v);
  }
}
template <>
__device__ inline void load4(const bf16* p, int64_t left, float (&v)[4]) {
  if (left >= 4) {
    const dc::u32x2_at2 w = __builtin_nontemporal_load(reinterpret_cast<const dc::u32x2_at2*>(p));
    v[0] = dc::bf16_lo(w.x), v[1] = dc::bf16_hi(w.x), v[2] = dc::bf16_lo(w.y), v[3] = dc::bf16_hi(w.y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? dc::to_f32(p[i]) : 0.0f;
  }
}
__device__ inline uint32_t load_codes(const uint8_t* p, int64_t left) {
  if (left >= 4) return __builtin_nontemporal_load(reinterpret_cast<const dc::u32_at1*>(p));
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) w |= (uint32_t)p[i] << (8 * i);
  return w;
}
__device__ inline void store_codes(uint8_t* p, int64_t left, uint32_t w) {
  if (left >= 4) {
    __builtin_nontemporal_store(w, reinterpret_cast<dc::u32_at1*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = (uint8_t)(w >> (8 * i));
  }
}
__device__ inline void store_copy(bf16* p, int64_t left, const float (&v)[4]) {
  if (left >= 4) {
    const dc::u32x2 w = {dc::pack_bf16(v[0], v[1]), dc::pack_bf16(v[2], v[3])};
    *reinterpret_cast<dc::u32x2_at2*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = dc::from_f32<bf16>(v[i]);
  }
}

// The block of 256 elements that is this wave's, from `start` on; a lane's four neighbouring ones of them.
template <bool kFp8, typename G>
__device__ inline void step_block(const Step& s, const Tensor& t, int64_t start) {
  const int lane = threadIdx.x & 63;
  const int64_t at = start + 4 * lane, left = t.n - at;
  float p[4] = {}, g[4] = {}, m[4] = {}, v[4] = {}, root[4];
  uint32_t mc = 0, vc = 0;
  float ms = 0.0f, vs = 0.0f;
  if (left > 0) {  // (all loads, then the arithmetic)
    load4(t.param + at, left, p);
    load4(static_cast<const G*>(t.grad) + at, left, g);
    if constexpr (kFp8) {
      mc = load_codes(static_cast<const uint8_t*>(t.m) + at, left);
      vc = load_codes(static_cast<const uint8_t*>(t.v) + at, left);
      ms = t.m_scales[at / kBlock];  // (the same for every lane; a scalar load would be waited for apart)
      vs = t.v_scales[at / kBlock];
    } else {
      load4(static_cast<const float*>(t.m) + at, left, m);
      load4(static_cast<const float*>(t.v) + at, left, v);
    }
  }
  if constexpr (kFp8) {
    unpack_fp8(mc, m);
    unpack_fp8(vc, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] *= ms;
      v[e] *= vs;
      v[e] *= v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float ge = g[e] * s.grad_scale;
    m[e] = s.beta1 * m[e] + s.rest1 * ge;
    v[e] = s.beta2 * v[e] + s.rest2 * (ge * ge);
    root[e] = sqrtf(v[e]);
    p[e] = p[e] * s.decay - s.rate * m[e] / (root[e] * s.root + s.eps);
  }
  if constexpr (kFp8) {  // (lanes past the tensor's end hold zeros)
    uint32_t mtop = 0, vtop = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mtop = max(mtop, dc::magnitude(m[e]));
      vtop = max(vtop, dc::magnitude(root[e]));
    }
    const float mt = __builtin_bit_cast(float, dc::wave_max_u32(mtop)), vt = __builtin_bit_cast(float, dc::wave_max_u32(vtop));
    const float mf = state_factor(mt), vf = state_factor(vt);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] *= mf;
      const float q = root[e] * vf;
      root[e] = root[e] > 0.0f && q < dc::kFp8Least ? dc::kFp8Least : q;
    }
    if (left > 0) {
      store_codes(static_cast<uint8_t*>(t.m) + at, left, dc::pack_fp8(m[0], m[1], m[2], m[3]));
      store_codes(static_cast<uint8_t*>(t.v) + at, left, dc::pack_fp8(root[0], root[1], root[2], root[3]));
      if (lane == 0) {
        t.m_scales[start / kBlock] = state_scale(mt);
        t.v_scales[start / kBlock] = state_scale(vt);
      }
    }
  } else if (left > 0) {
    store4(static_cast<float*>(t.m) + at, left, m);
    store4(static_cast<float*>(t.v) + at, left, v);
  }
  if (left > 0) {
    store4(t.param + at, left, p);
    if (t.copy) store_copy(reinterpret_cast<bf16*>(t.copy) + at, left, p);
  }
}

// The tensor of a chunk is the last whose first chunk is not past it. In a short launch, which is latency, a wave's lanes
// compare one each, a single load; in a long one bisection, whose scalar loads hit and cost the vector units nothing. Measured, us, lanes /
// bisection: 484 thousand elements in 30 tensors 4.5 / 5.0, 8-bit states 4.8 / 5.7; 12 million in 10, 8-bit, 31.8 / 32.3; 134 million
// in 20, 8-bit, 382 / 369.
constexpr int64_t kLongLaunch = 32768;  // chunks
template <bool kFp8, bool kLong>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Step s) {
  const uint32_t chunk = blockIdx.x;
  int lo = 0;
  if constexpr (kLong) {
    for (int hi = s.count; hi - lo > 1;) {
      const int mid = (lo + hi) >> 1;
      if (s.first[mid] <= chunk) lo = mid;
      else hi = mid;
    }
  } else {
    const int lane = threadIdx.x & 63;
    const uint32_t first = s.first[lane < kTensors ? lane : kTensors - 1];
    lo = __popcll(__ballot(lane < s.count && first <= chunk)) - 1;
  }
  const Tensor& t = s.t[lo];
  const int64_t start = (int64_t)(chunk - s.first[lo]) * kChunk + (threadIdx.x >> 6) * kBlock;
  if (t.grad_f32) step_block<kFp8, float>(s, t, start);
  else step_block<kFp8, bf16>(s, t, start);
}

bool aligned_to(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int32_t check_tensor(const dc_adamw_tensor& t, bool fp8) {
  if (t.n < 0 || t.reserved != 0) return DC_ERR_INVALID_ARGUMENT;
  if (t.grad_dtype != DC_DTYPE_F32 && t.grad_dtype != DC_DTYPE_BF16) return DC_ERR_INVALID_ARGUMENT;
  if (!fp8 && (t.m_scales || t.v_scales)) return DC_ERR_INVALID_ARGUMENT;
  if (t.n == 0) return DC_OK;
  if (!t.param || !t.grad || !t.m || !t.v || (fp8 && (!t.m_scales || !t.v_scales))) return DC_ERR_INVALID_ARGUMENT;
  const bool ok = aligned_to(t.param, 4) && aligned_to(t.grad, t.grad_dtype == DC_DTYPE_F32 ? 4 : 2) &&
                  aligned_to(t.copy, 2) && aligned_to(t.m_scales, 4) && aligned_to(t.v_scales, 4) &&
                  (fp8 || (aligned_to(t.m, 4) && aligned_to(t.v, 4)));
  return ok ? DC_OK : DC_ERR_MISALIGNED;
}

constexpr int64_t kMaxPiece = int64_t(1) << 33;    // elements of a tensor's part in one launch
constexpr int64_t kMaxChunks = int64_t(1) << 23;   // of a launch (2^31 work items)
static_assert(kMaxPiece % kBlock == 0 && kMaxPiece / kChunk <= kMaxChunks);

}  // namespace

extern "C" DC_HIP_API int32_t dc_hip_adamw_step(dc_hip_ctx* ctx, const dc_adamw* args, const dc_adamw_tensor* tensors,
                                                int32_t count) {
  if (!args || count < 0 || (count > 0 && !tensors)) return DC_ERR_INVALID_ARGUMENT;
  const dc_adamw& a = *args;
  const bool fp8 = a.state_dtype == DC_DTYPE_FP8;
  if ((!fp8 && a.state_dtype != DC_DTYPE_F32) || a.reserved != 0 || a.step < 1) return DC_ERR_INVALID_ARGUMENT;
  if (!(a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0 && a.eps >= 0.0) || !std::isfinite(a.lr) ||
      !std::isfinite(a.weight_decay) || !std::isfinite(a.grad_scale))
    return DC_ERR_INVALID_ARGUMENT;
  for (int32_t i = 0; i < count; ++i) DC_RETURN_IF(check_tensor(tensors[i], fp8));
  DC_CTX_ENTER(ctx);
  Step s;
  s.beta1 = (float)a.beta1, s.beta2 = (float)a.beta2;
  s.rest1 = (float)(1.0 - a.beta1), s.rest2 = (float)(1.0 - a.beta2);
  s.rate = (float)(a.lr / (1.0 - std::pow(a.beta1, (double)a.step)));
  s.root = (float)(1.0 / std::sqrt(1.0 - std::pow(a.beta2, (double)a.step)));
  s.eps = (float)a.eps, s.decay = (float)(1.0 - a.lr * a.weight_decay), s.grad_scale = (float)a.grad_scale;
  s.count = 0;
  int64_t chunks = 0;
  auto launch = [&]() -> int32_t {
    if (s.count == 0) return DC_OK;
    const bool longer = chunks > kLongLaunch;
    const unsigned grid = (unsigned)chunks;
    if (fp8 && longer) adamw_kernel<true, true><<<grid, kThreads, 0, ctx->stream>>>(s);
    else if (fp8) adamw_kernel<true, false><<<grid, kThreads, 0, ctx->stream>>>(s);
    else if (longer) adamw_kernel<false, true><<<grid, kThreads, 0, ctx->stream>>>(s);
    else adamw_kernel<false, false><<<grid, kThreads, 0, ctx->stream>>>(s);
    s.count = 0;
    chunks = 0;
    return dc::last_launch_status();
  };
  for (int32_t i = 0; i < count; ++i) {
    const dc_adamw_tensor& t = tensors[i];
    const int64_t grad_size = t.grad_dtype == DC_DTYPE_F32 ? 4 : 2, state_size = fp8 ? 1 : 4;
    for (int64_t off = 0; off < t.n; off += kMaxPiece) {
      const int64_t n = std::min(t.n - off, kMaxPiece), more = (n + kChunk - 1) / kChunk;
      if (s.count == kTensors || chunks + more > kMaxChunks) DC_RETURN_IF(launch());
      s.first[s.count] = (uint32_t)chunks;
      s.t[s.count++] = Tensor{t.param + off,
                              static_cast<const char*>(t.grad) + off * grad_size,
                              static_cast<char*>(t.m) + off * state_size,
                              static_cast<char*>(t.v) + off * state_size,
                              fp8 ? t.m_scales + off / kBlock : nullptr,
                              fp8 ? t.v_scales + off / kBlock : nullptr,
                              t.copy ? t.copy + off : nullptr,
                              n,
                              t.grad_dtype == DC_DTYPE_F32};
      chunks += more;
    }
  }
  return launch();
}
