// One AdamW step over many tensors:
//     m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        t = t + 1
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// in fp32 whatever the parameters' and gradients' type; a parameter in 16 bits is rounded to nearest once, as it is stored.
//
// Bound by HBM: p, g, m and v are read and p, m, v written once, 28 bytes a parameter in fp32.  With moments in 8 bits it is 16.
// Measured for 38 M parameters in 188 tensors, fp32: 170 us, 6.2 TB/s, with moments in 32 bits; 165 us with 8 bits, where the
// integer pipe is 64 % busy with hashes and codes and 550 MB of HBM traffic are not the limit (decoding both moments: 57 us).
//
// 8-bit moments are codes of a logarithmic scale: the code k > 0 of a block of 256 elements stands for the fp32 number with the
// bits (k + base) << 20, i.e. 8 values to an octave, the code 0 for zero.  The block's base puts its largest magnitude at the
// last code but one; 127 codes and a sign (m) span 16 octaves below it, 255 codes (v) 32, as many as the squares of m's.  An
// addition and a shift of the fp32 bits are the whole conversion, and a block's scale needs a maximum of integers and no division.
// Numbers are rounded to one of their two neighbours at random: v moves by a thousandth per step, an eighth of a thousandth of
// the codes' spacing, and rounding to nearest would never move it.  The random bits are a hash of the tensor's step and the
// element's place, so that a step repeated from the same state gives the same bits.  A second moment that is not zero never
// becomes zero (it is the divisor of a first moment that may not have); a first moment below the first code becomes that or zero.
// The updates of m and v are single roundings in a fixed order (no contraction), as the codes go by the last bit.
//
// A warp works on 256 elements, a code block; a lane has eight consecutive ones, whose loads (p, g, m, v) are all in flight at
// once.  The tensors' addresses travel in the kernel's parameters (no copy to the device); a block finds its tensor by bisection.
// The last block to have read the steps writes them, advanced: nothing of a step is on the host, so it can be captured and a
// step that `found_inf` cancels leaves everything as it was.
#include <math.h>
#include <string.h>

#include "wcn_common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int CODES = 256;                                   // elements of a code block: a warp's
constexpr int CHUNK = THREADS / 32 * CODES;                  // elements of a thread block
constexpr int FEW = 48, SOME = 240, MANY = 640;              // tensors of a launch: 2, 10 and 26 KB of parameters

struct Tensor {
  void* param;
  const void* grad;
  int64_t n;
  int64_t slot;        // first element of its moments, a multiple of CODES
  int32_t step;        // its place in `steps`
  int32_t first;       // first thread block
};

template <int MAX> struct Table { Tensor t[MAX]; };

struct Hyper {
  int count;
  void* m;
  void* v;
  int16_t* m_base;
  int16_t* v_base;
  int32_t* steps;
  const float* lr_at;        // learning rate on the device (or null)
  const float* grad_scale;   // gradients are divided by it (or null)
  const float* found_inf;    // not zero: the step is cancelled (or null)
  unsigned* counter;
  float lr, wd, eps, b1, b1c, b2, b2c, log_b1, log_b2;
};

// Eight elements of a lane; fp32 ones in one request of 32 bytes (two of 16 touch every line twice).
template <typename T> __device__ __forceinline__ void load8(const T* p, int64_t left, bool vec, float (&x)[8]) {
  if (vec && left >= 8) {
    __align__(32) T v[8];
    if constexpr (sizeof(T) == 4) {
      asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]) : "l"(p));
    } else {
      *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = wcn_to_float<T>(v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < left ? wcn_to_float<T>(p[i]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, int64_t left, bool vec, const float (&x)[8]) {
  if (vec && left >= 8) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]),
                   "f"(x[5]), "f"(x[6]), "f"(x[7]) : "memory");
    } else {
      __align__(16) T v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = wcn_from_float<T>(x[i]);
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = wcn_from_float<T>(x[i]);
  }
}

// m / (sqrt(v) * root + eps), to one part in 2^21 of an update.  (Second moments below 2^-126 are numbers: gradients of 1e-18 have
// such ones, and with an epsilon below them an update as large as any.)
__device__ __forceinline__ float quotient(float m, float v, float root, float eps) {
  float s, r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(s) : "f"(v));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(s, root, eps)));
  return m * r;
}

__device__ __forceinline__ float code_value(uint32_t k, uint32_t base) { return k ? __uint_as_float((k + base) << 20) : 0.f; }

// The base of a block whose largest magnitude has these bits, and what a rounded number may become at most: numbers stay
// numbers, and NaN (whose payload an addition could carry past the end) NaN.
__device__ __forceinline__ uint32_t code_base(uint32_t top_bits, uint32_t codes) {
  const uint32_t q = (top_bits >> 20) + 1;
  return q > codes ? q - codes : 0;
}
__device__ __forceinline__ uint32_t code_limit(uint32_t top_bits) { return top_bits < 0x7F800000u ? 0x7F7u : 0x7FFu; }

// Codes of a lane's eight numbers (bits of the magnitudes), one a byte, given 20 random bits for each.  `signs`: the first
// moment, whose sign is the code's top bit.
template <bool SIGNS> __device__ __forceinline__ uint2 pack8(const float (&x)[8], const uint32_t (&random)[8], uint32_t base, uint32_t top_bits) {
  uint32_t k[8];
  bool low = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = __float_as_uint(x[i]) & 0x7FFFFFFFu, q = (bits + random[i]) >> 20;
    k[i] = q - base;
    if (SIGNS) low |= q <= base;
    else k[i] = bits ? (uint32_t)max((int)k[i], 1) : 0u;
  }
  // rare, and the same for a warp: numbers below the first code (first moment), numbers near the end of fp32
  if (SIGNS && base && __any_sync(0xFFFFFFFFu, low)) {
    const float first = __uint_as_float((base + 1) << 20);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = __float_as_uint(x[i]) & 0x7FFFFFFFu;
      if (((bits + random[i]) >> 20) <= base) k[i] = __uint_as_float(bits) > __fmul_rn(first, __fmul_rn((float)random[i], 9.5367431640625e-7f)) ? 1 : 0;   // 2^-20
    }
  }
  if (top_bits >= 0x7F600000u) {
    const uint32_t most = code_limit(top_bits) - base;
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] = min(k[i], most);
  }
  if (SIGNS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) k[i] |= (__float_as_uint(x[i]) >> 24) & 128u;
  }
  auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410); };
  return make_uint2(four(k[0], k[1], k[2], k[3]), four(k[4], k[5], k[6], k[7]));
}

template <typename P, typename G, bool EIGHT, int MAX>
__global__ void __launch_bounds__(THREADS) adamw_kernel(const __grid_constant__ Table<MAX> table, const __grid_constant__ Hyper h) {
  __shared__ float factors[3];
  __shared__ uint32_t salt;
  if (h.found_inf && *h.found_inf != 0.f) return;
  int at = 0;
  for (int hi = h.count; hi - at > 1;) {
    const int mid = (at + hi) / 2;
    if (table.t[mid].first <= (int)blockIdx.x) at = mid; else hi = mid;
  }
  const Tensor& t = table.t[at];
  const int64_t e = (int64_t)((int)blockIdx.x - t.first) * CHUNK + threadIdx.x * 8;
  const int64_t left = t.n - e;                              // of this lane's elements on
  const bool mine = left + (threadIdx.x & 31) * 8 > 0;       // the warp's block has an element of the tensor
  const int64_t s = t.slot + e;
  P* const param = reinterpret_cast<P*>(t.param) + e;
  const G* const grad = reinterpret_cast<const G*>(t.grad) + e;
  const bool pvec = reinterpret_cast<uintptr_t>(t.param) % (8 * sizeof(P)) == 0, gvec = reinterpret_cast<uintptr_t>(t.grad) % (8 * sizeof(G)) == 0;

  float p[8], g[8], m[8], v[8];
  if (mine) {
    load8<P>(param, left, pvec, p);
    load8<G>(grad, left, gvec, g);
    if (EIGHT) {
      const uint2 cm = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(h.m) + s);
      const uint2 cv = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(h.v) + s);
      const uint32_t mb = (uint32_t)(int)h.m_base[s / CODES], vb = (uint32_t)(int)h.v_base[s / CODES];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t km = ((i < 4 ? cm.x : cm.y) >> (i % 4 * 8)) & 255u, kv = ((i < 4 ? cv.x : cv.y) >> (i % 4 * 8)) & 255u;
        m[i] = code_value(km & 127u, mb);
        m[i] = km & 128u ? -m[i] : m[i];
        v[i] = code_value(kv, vb);
      }
    } else {
      load8<float>(reinterpret_cast<const float*>(h.m) + s, 8, true, m);
      load8<float>(reinterpret_cast<const float*>(h.v) + s, 8, true, v);
    }
  }
  if (threadIdx.x == 0) {
    const int now = h.steps[t.step] + 1;
    const float lr = h.lr_at ? *h.lr_at : h.lr;
    factors[0] = lr / -expm1f((float)now * h.log_b1);        // lr / (1 - b1^t)
    factors[1] = rsqrtf(-expm1f((float)now * h.log_b2));     // 1 / sqrt(1 - b2^t)
    factors[2] = 1.f - lr * h.wd;
    salt = wcn_fmix32((uint32_t)now);
  }
  __syncthreads();
  if (threadIdx.x == 0) {                                    // (this block has read its step)
    __threadfence();
    if (atomicAdd(h.counter, 1u) == gridDim.x - 1) {
      *h.counter = 0;
      for (int i = 0; i < h.count; ++i) h.steps[table.t[i].step] += 1;
    }
  }
  if (!mine) return;
  const float size = factors[0], root = factors[1], keep = factors[2], inv = h.grad_scale ? 1.f / *h.grad_scale : 1.f;
  uint32_t m_top = 0, v_top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = h.grad_scale ? g[i] * inv : g[i];
    m[i] = __fadd_rn(__fmul_rn(m[i], h.b1), __fmul_rn(d, h.b1c));
    v[i] = __fadd_rn(__fmul_rn(v[i], h.b2), __fmul_rn(__fmul_rn(d, d), h.b2c));
    p[i] = p[i] * keep - size * quotient(m[i], v[i], root, h.eps);
    m_top = max(m_top, __float_as_uint(m[i]) & 0x7FFFFFFFu);
    v_top = max(v_top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  }
  if (left > 0) store8<P>(param, left, pvec, p);
  if (EIGHT) {
    m_top = __reduce_max_sync(0xFFFFFFFFu, m_top);
    v_top = __reduce_max_sync(0xFFFFFFFFu, v_top);
    const uint32_t mb = code_base(m_top, 127), vb = code_base(v_top, 255);
    uint32_t for_m[8], for_v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t random = wcn_fmix32((uint32_t)(s + i) * 0x9E3779B9u ^ salt);
      for_m[i] = random >> 12;
      for_v[i] = (random * 0x9E3779B1u) >> 12;
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(h.m) + s) = pack8<true>(m, for_m, mb, m_top);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(h.v) + s) = pack8<false>(v, for_v, vb, v_top);
    if ((threadIdx.x & 31) == 0) {
      h.m_base[s / CODES] = (int16_t)mb;
      h.v_base[s / CODES] = (int16_t)vb;
    }
  } else {
    store8<float>(reinterpret_cast<float*>(h.m) + s, 8, true, m);
    store8<float>(reinterpret_cast<float*>(h.v) + s, 8, true, v);
  }
}

// The numbers that codes stand for: eight of each moment a thread.
__global__ void __launch_bounds__(THREADS) decode_moments_kernel(const uint8_t* m, const int16_t* m_base, const uint8_t* v,
                                                                 const int16_t* v_base, int64_t n, float* m_out, float* v_out) {
  const int64_t s = ((int64_t)blockIdx.x * THREADS + threadIdx.x) * 8;
  if (s >= n) return;
  const uint2 cm = __ldg(reinterpret_cast<const uint2*>(m + s)), cv = __ldg(reinterpret_cast<const uint2*>(v + s));
  const uint32_t mb = (uint32_t)(int)__ldg(&m_base[s / CODES]), vb = (uint32_t)(int)__ldg(&v_base[s / CODES]);
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t km = ((i < 4 ? cm.x : cm.y) >> (i % 4 * 8)) & 255u, kv = ((i < 4 ? cv.x : cv.y) >> (i % 4 * 8)) & 255u;
    x[i] = code_value(km & 127u, mb);
    x[i] = km & 128u ? -x[i] : x[i];
    y[i] = code_value(kv, vb);
  }
  store8<float>(m_out + s, 8, true, x);
  store8<float>(v_out + s, 8, true, y);
}

template <typename P, typename G, bool EIGHT, int MAX>
int launch(const Tensor* t, Hyper& h, int count, unsigned blocks, cudaStream_t st) {
  Table<MAX> table;
  memcpy(table.t, t, sizeof(Tensor) * count);
  h.count = count;
  adamw_kernel<P, G, EIGHT, MAX><<<blocks, THREADS, 0, st>>>(table, h);
  ++wcn_launched;
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}

// What a call is given of its tensors.
struct Given {
  const int64_t *params, *grads, *sizes, *slots, *step_at;   // slots, step_at: null: one after the other
  int64_t count;
};

template <typename P, typename G, bool EIGHT>
int run(const Given& a, Hyper& h, cudaStream_t st) {
  Tensor t[MANY];
  int64_t slot = 0;
  for (int64_t i = 0; i < a.count;) {
    int k = 0;
    int64_t blocks = 0;
    for (; i < a.count && k < MANY; ++i) {
      const int64_t n = a.sizes[i], need = (n + CHUNK - 1) / CHUNK;
      if (blocks + need > 0x7FFFFFFF) break;
      if (need) t[k++] = {(void*)a.params[i], (const void*)a.grads[i], n, a.slots ? a.slots[i] : slot, (int32_t)(a.step_at ? a.step_at[i] : i), (int32_t)blocks};
      blocks += need;
      slot += (n + CODES - 1) / CODES * CODES;
    }
    if (!k) {
      if (i < a.count) return WCN_ERR_INVALID_PARAMETERS;    // (one tensor of 2^42 elements)
      break;
    }
    const int rc = k <= FEW ? launch<P, G, EIGHT, FEW>(t, h, k, (unsigned)blocks, st) : k <= SOME ? launch<P, G, EIGHT, SOME>(t, h, k, (unsigned)blocks, st)
                                                                                                   : launch<P, G, EIGHT, MANY>(t, h, k, (unsigned)blocks, st);
    if (rc != WCN_OK) return rc;
  }
  return WCN_OK;
}

template <typename P, bool EIGHT>
int by_grad(int dtype, const Given& a, Hyper& h, cudaStream_t st) {
  if (dtype == WCN_F32) return run<P, float, EIGHT>(a, h, st);
  if (dtype == WCN_F16) return run<P, __half, EIGHT>(a, h, st);
  return run<P, __nv_bfloat16, EIGHT>(a, h, st);
}

template <bool EIGHT>
int by_param(int dtype, int grad_dtype, const Given& a, Hyper& h, cudaStream_t st) {
  if (dtype == WCN_F32) return by_grad<float, EIGHT>(grad_dtype, a, h, st);
  if (dtype == WCN_F16) return by_grad<__half, EIGHT>(grad_dtype, a, h, st);
  return by_grad<__nv_bfloat16, EIGHT>(grad_dtype, a, h, st);
}

bool on32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

double number(int64_t bits) {
  double d;
  memcpy(&d, &bits, sizeof d);
  return d;
}

}  // namespace

extern "C" int wcn_adamw_step(const int64_t* params, const int64_t* grads, const int64_t* sizes, const int64_t* slots,
                              const int64_t* step_at, int64_t count, int dtype, int grad_dtype, void* exp_avg, int16_t* exp_avg_base,
                              void* exp_avg_sq, int16_t* exp_avg_sq_base, int64_t length, int32_t* steps, int64_t num_steps,
                              int64_t lr_bits, int64_t beta1_bits, int64_t beta2_bits, int64_t eps_bits, int64_t weight_decay_bits,
                              const float* lr, const float* grad_scale, const float* found_inf, uint32_t* counter, void* stream) {
  wcn_launched = 0;
  if (count < 0 || (count && (!params || !grads || !sizes || !counter || (length && (!exp_avg || !exp_avg_sq)) || (num_steps && !steps))) || dtype < WCN_F32 ||
      dtype > WCN_BF16 || grad_dtype < WCN_F32 || grad_dtype > WCN_BF16 || !on32(exp_avg) || !on32(exp_avg_sq) || !exp_avg_base != !exp_avg_sq_base)
    return WCN_ERR_INVALID_PARAMETERS;
  const double b1 = number(beta1_bits), b2 = number(beta2_bits);
  if (!(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1)) return WCN_ERR_INVALID_PARAMETERS;
  int64_t slot = 0;
  for (int64_t i = 0; i < count; ++i) {
    const int64_t n = sizes[i], at = step_at ? step_at[i] : i;
    if (slots) slot = slots[i];
    if (n < 0 || (n && (!params[i] || !grads[i])) || params[i] % wcn_dtype_size(dtype) || grads[i] % wcn_dtype_size(grad_dtype) || slot < 0 ||
        slot % CODES || at < 0 || at > 0x7FFFFFFF)
      return WCN_ERR_INVALID_PARAMETERS;
    // (in blocks: the sum of a slot and a size may be beyond 63 bits)
    const int64_t end = slot / CODES + n / CODES + (n % CODES != 0);
    if (end > length / CODES || at >= num_steps) return WCN_ERR_BOUNDS;
    slot = end * CODES;
  }
  const Given a = {params, grads, sizes, slots, step_at, count};
  Hyper h = {};
  h.m = exp_avg; h.v = exp_avg_sq; h.m_base = exp_avg_base; h.v_base = exp_avg_sq_base; h.steps = steps;
  h.lr_at = lr; h.grad_scale = grad_scale; h.found_inf = found_inf; h.counter = counter;
  h.lr = (float)number(lr_bits); h.wd = (float)number(weight_decay_bits); h.eps = (float)number(eps_bits);
  h.b1 = (float)b1; h.b1c = (float)(1 - b1); h.b2 = (float)b2; h.b2c = (float)(1 - b2);
  h.log_b1 = (float)log(b1); h.log_b2 = (float)log(b2);
  cudaStream_t st = wcn_stream(stream);
  return exp_avg_base ? by_param<true>(dtype, grad_dtype, a, h, st) : by_param<false>(dtype, grad_dtype, a, h, st);
}

extern "C" int wcn_adamw_decode(const void* exp_avg, const int16_t* exp_avg_base, const void* exp_avg_sq,
                                const int16_t* exp_avg_sq_base, int64_t n, float* exp_avg_out, float* exp_avg_sq_out, void* stream) {
  if (n < 0 || n % CODES || n / CODES > 0x7FFFFFFFll) return WCN_ERR_INVALID_PARAMETERS;
  if (!n) return WCN_OK;
  if (!exp_avg || !exp_avg_sq || !exp_avg_base || !exp_avg_sq_base || !exp_avg_out || !exp_avg_sq_out || !on32(exp_avg) ||
      !on32(exp_avg_sq) || !on32(exp_avg_out) || !on32(exp_avg_sq_out))
    return WCN_ERR_INVALID_PARAMETERS;
  const int64_t blocks = (n + THREADS * 8 - 1) / (THREADS * 8);
  decode_moments_kernel<<<(unsigned)blocks, THREADS, 0, wcn_stream(stream)>>>((const uint8_t*)exp_avg, exp_avg_base, (const uint8_t*)exp_avg_sq,
                                                                            exp_avg_sq_base, n, exp_avg_out, exp_avg_sq_out);
  return cudaGetLastError() == cudaSuccess ? WCN_OK : WCN_ERR_EXECUTION;
}
