// dc_adamw.hip — one AdamW step over many tensors at once, states in 32 bits or in 8 bits with scales.
//
// Memory-bound: an element with 32-bit states moves 28 bytes (gradient 2; param, m, v in and out 24; the bf16 copy 2),
// with 8-bit ones 16. The tensors' addresses travel in the kernel's arguments, kTensors a launch, so a step of a whole
// model is a few launches, nothing is uploaded and nothing is kept between calls. A workgroup takes kChunk elements of one
// tensor (found by bisection over the tensors' first chunks, in scalar registers); a wave's 64 lanes take 4 neighbouring
// elements each, which is one 8-bit state block: its maximum is a DPP reduction, and a state's codes and scale are read
// and written once.
#include <algorithm>
#include <cmath>

#include "dc_internal.hpp"
#include "dc_numeric.hpp"

namespace {

using dc::bf16;

constexpr int kTensors = 48;  // of a launch: their table, 3.5 KiB, travels in the kernel's arguments
constexpr int kThreads = 256;
constexpr int kBlock = DC_ADAMW_BLOCK;
constexpr int kRounds = 4;  // blocks of a wave
constexpr int kChunk = kThreads / 64 * kBlock * kRounds;
static_assert(kBlock == 64 * 4, "a wave's lanes take four elements each of a block");

struct Tensor {
  float* param;
  const void* grad;
  void *m, *v;
  float *m_scales, *v_scales;
  uint16_t* copy;
  int64_t n;
  uint32_t first;  // of its chunks in the launch
  int32_t grad_f32;
};

struct Step {
  float beta1, beta2, rest1, rest2;  // rest: 1 - beta
  float rate, root, eps, decay;      // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), eps, 1 - lr weight_decay
  float grad_scale;
  int32_t count;
  Tensor t[kTensors];
};

// Four 8-bit states with their scale.
__device__ inline void unpack_fp8(uint32_t w, float (&v)[4]) {
  const dc::f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
}

// The elements [0, 4) at p of which `left` exist; zeros for the others.
template <typename T>
__device__ inline void load4(const T* p, int64_t left, float (&v)[4]);
template <>
__device__ inline void load4(const float* p, int64_t left, float (&v)[4]) {
  dc::load_some(p, left, v);
}
template <>
__device__ inline void load4(const bf16* p, int64_t left, float (&v)[4]) {
  if (left >= 4) {
    const dc::u32x2_at2 w = *reinterpret_cast<const dc::u32x2_at2*>(p);
    v[0] = dc::bf16_lo(w.x), v[1] = dc::bf16_hi(w.x), v[2] = dc::bf16_lo(w.y), v[3] = dc::bf16_hi(w.y);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? dc::to_f32(p[i]) : 0.0f;
  }
}
__device__ inline uint32_t load_codes(const uint8_t* p, int64_t left) {
  if (left >= 4) return *reinterpret_cast<const dc::u32_at1*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) w |= (uint32_t)p[i] << (8 * i);
  return w;
}
__device__ inline void store_codes(uint8_t* p, int64_t left, uint32_t w) {
  if (left >= 4) {
    *reinterpret_cast<dc::u32_at1*>(p) = w;
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

template <bool kFp8, typename G>
__device__ inline void step_chunk(const Step& s, const Tensor& t, int64_t start) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float p[kRounds][4], g[kRounds][4], m[kRounds][4], v[kRounds][4];
  uint32_t mc[kRounds], vc[kRounds];
  float ms[kRounds], vs[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {  // all loads of the chunk, then the arithmetic
    const int64_t at = start + ((int64_t)i * (kThreads / 64) + wave) * kBlock + 4 * lane, left = t.n - at;
    if (left > 0) {
      load4(t.param + at, left, p[i]);
      load4(static_cast<const G*>(t.grad) + at, left, g[i]);
      if constexpr (kFp8) {
        mc[i] = load_codes(static_cast<const uint8_t*>(t.m) + at, left);
        vc[i] = load_codes(static_cast<const uint8_t*>(t.v) + at, left);
        ms[i] = t.m_scales[at / kBlock];
        vs[i] = t.v_scales[at / kBlock];
      } else {
        load4(static_cast<const float*>(t.m) + at, left, m[i]);
        load4(static_cast<const float*>(t.v) + at, left, v[i]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) p[i][e] = g[i][e] = m[i][e] = v[i][e] = 0.0f;
      mc[i] = vc[i] = 0;
      ms[i] = vs[i] = 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int64_t at = start + ((int64_t)i * (kThreads / 64) + wave) * kBlock + 4 * lane, left = t.n - at;
    if constexpr (kFp8) {
      unpack_fp8(mc[i], m[i]);
      unpack_fp8(vc[i], v[i]);
    }
    float root[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (kFp8) {
        m[i][e] *= ms[i];
        v[i][e] *= vs[i];
        v[i][e] *= v[i][e];
      }
      const float ge = g[i][e] * s.grad_scale;
      m[i][e] = s.beta1 * m[i][e] + s.rest1 * ge;
      v[i][e] = s.beta2 * v[i][e] + s.rest2 * (ge * ge);
      root[e] = sqrtf(v[i][e]);
      p[i][e] = p[i][e] * s.decay - s.rate * m[i][e] / (root[e] * s.root + s.eps);
    }
    if constexpr (kFp8) {
      // (a wave's lanes hold one block; those past its end hold zeros)
      uint32_t mtop = 0, vtop = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mtop = max(mtop, dc::magnitude(m[i][e]));
        vtop = max(vtop, dc::magnitude(root[e]));
      }
      const float mt = __builtin_bit_cast(float, dc::wave_max_u32(mtop)), vt = __builtin_bit_cast(float, dc::wave_max_u32(vtop));
      const float mf = dc::fp8_factor(mt), vf = dc::fp8_factor(vt);
      float mq[4], vq[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mq[e] = m[i][e] * mf;
        vq[e] = root[e] * vf;
        if (root[e] > 0.0f && vq[e] < dc::kFp8Least) vq[e] = dc::kFp8Least;
      }
      if (left > 0) {
        store_codes(static_cast<uint8_t*>(t.m) + at, left, dc::pack_fp8(mq[0], mq[1], mq[2], mq[3]));
        store_codes(static_cast<uint8_t*>(t.v) + at, left, dc::pack_fp8(vq[0], vq[1], vq[2], vq[3]));
        if (lane == 0) {
          t.m_scales[at / kBlock] = mt / dc::kFp8Top;
          t.v_scales[at / kBlock] = vt / dc::kFp8Top;
        }
      }
    } else if (left > 0) {
      dc::store_some(static_cast<float*>(t.m) + at, left, m[i]);
      dc::store_some(static_cast<float*>(t.v) + at, left, v[i]);
    }
    if (left > 0) {
      dc::store_some(t.param + at, left, p[i]);
      if (t.copy) store_copy(reinterpret_cast<bf16*>(t.copy) + at, left, p[i]);
    }
  }
}

template <bool kFp8>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Step s) {
  const uint32_t chunk = blockIdx.x;
  int lo = 0, hi = s.count;  // the last tensor whose first chunk is not past this one
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s.t[mid].first <= chunk) lo = mid;
    else hi = mid;
  }
  const Tensor& t = s.t[lo];
  const int64_t start = (int64_t)(chunk - t.first) * kChunk;
  if (t.grad_f32) step_chunk<kFp8, float>(s, t, start);
  else step_chunk<kFp8, bf16>(s, t, start);
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

constexpr int64_t kMaxPiece = int64_t(1) << 34;    // elements of a tensor's part in one launch
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
    if (fp8) adamw_kernel<true><<<(unsigned)chunks, kThreads, 0, ctx->stream>>>(s);
    else adamw_kernel<false><<<(unsigned)chunks, kThreads, 0, ctx->stream>>>(s);
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
      s.t[s.count++] = Tensor{t.param + off,
                              static_cast<const char*>(t.grad) + off * grad_size,
                              static_cast<char*>(t.m) + off * state_size,
                              static_cast<char*>(t.v) + off * state_size,
                              fp8 ? t.m_scales + off / kBlock : nullptr,
                              fp8 ? t.v_scales + off / kBlock : nullptr,
                              t.copy ? t.copy + off : nullptr,
                              n,
                              (uint32_t)chunks,
                              t.grad_dtype == DC_DTYPE_F32};
      chunks += more;
    }
  }
  return launch();
}
