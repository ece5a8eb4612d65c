// logits.cu - what a model may answer with, and what it learns from: penalties,
// biases and masks on rows of logits, and the masked softmax cross entropy
// with its gradient.  Rows are [vocab] of fp32, bf16 or fp16 at any stride;
// arithmetic is fp32, rounded once at the store.
#include <algorithm>

#include "rowvec.cuh"

namespace cnnue {
namespace logits {
namespace {

using rows::kNegInf;
using rows::Vec;

constexpr int64_t kMaxVocab = (int64_t)1 << 30;  // element offsets inside a row are 32-bit

// ---------------------------------------------------------------------------
// Penalties, biases, masks.
//
//   x = l
//   seen in the history:   x = x > 0 ? x / repetition : x * repetition
//   c = its count in the part after the prompt:
//                          x = x - frequency * c;  x = x - presence  (c > 0)
//   x = x + bias            for the token's biases in list order
//   not allowed:           x = -inf
//
// Every step is one IEEE fp32 operation.  A CTA takes one slice of one row: it
// counts the history's tokens that fall into the slice in shared memory
// (integer atomics: their order does not change the counts), marks the
// slice's biased tokens, and then streams the slice.
// ---------------------------------------------------------------------------

constexpr int kProcThreads = 256;
constexpr uint32_t kSeen = 0x80000000u;     // counter: the token occurs (prompt or not); low bits: its count
constexpr uint32_t kNoBias = 0x7fffffffu;   // bias slot: no entry; else the first entry's position,
constexpr uint32_t kRepeated = 0x80000000u; // with this bit when more entries name the token

struct ProcArgs {
  const void* in;
  void* out;
  int64_t in_stride, out_stride;
  int vocab, split, vps;  // slices per row, vectors per slice
  cnnue_logit_rules r;
  uint32_t* status;
};

template <typename TI, typename TO, bool HIST, bool BIAS>
__global__ void __launch_bounds__(kProcThreads) process_kernel(const ProcArgs a) {
  constexpr int VE = Vec<TI>::VE;
  extern __shared__ uint32_t slots[];
  const int64_t row = blockIdx.x / a.split;
  const int part = (int)(blockIdx.x % a.split);
  const TI* in = (const TI*)a.in + row * a.in_stride;
  TO* out = (TO*)a.out + row * a.out_stride;
  const int shift = rows::shift_of(in);
  const int v0 = part * a.vps;
  const int lo = v0 * VE - shift;  // first token of the slice
  const int width = a.vps * VE;    // tokens per slice
  uint32_t* count = slots;
  uint32_t* first = slots + (HIST ? width : 0);

  bool dead = false;  // the row's mask index is out of range: nothing is allowed
  const uint32_t* mask = nullptr;
  if (a.r.mask) {
    const int64_t m = a.r.mask_index ? (int64_t)a.r.mask_index[row] : a.r.mask_rows == 1 ? 0 : row;
    if (m >= a.r.mask_rows) {
      dead = true;
      if (threadIdx.x == 0 && part == 0) atomicOr(a.status, CNNUE_STATUS_BAD_INDEX);
    } else if (m >= 0) {
      mask = a.r.mask + m * a.r.mask_stride;
    }
  }

  float rep = 1.f, freq = 0.f, pres = 0.f;
  const int32_t* btok = nullptr;
  const float* bval = nullptr;
  if (HIST || BIAS) {
    for (int i = threadIdx.x; i < width; i += kProcThreads) {
      if (HIST) count[i] = 0;
      if (BIAS) first[i] = kNoBias;
    }
    __syncthreads();
  }
  if (HIST) {
    if (a.r.repetition) rep = a.r.repetition[row];
    if (a.r.frequency) freq = a.r.frequency[row];
    if (a.r.presence) pres = a.r.presence[row];
    int64_t len = a.r.history_len;
    if (a.r.lengths) {
      const int64_t l = a.r.lengths[row];
      if (l < 0 || l > len) {
        if (threadIdx.x == 0 && part == 0) atomicOr(a.status, CNNUE_STATUS_BAD_OFFSETS);
        len = l < 0 ? 0 : len;
      } else {
        len = l;
      }
    }
    const int64_t prompt = a.r.prompt_lengths ? a.r.prompt_lengths[row] : 0;
    const bool wide = a.r.history_bytes == 8;
    const char* list = (const char*)a.r.history + row * a.r.history_stride * a.r.history_bytes;
    for (int64_t i = threadIdx.x; i < len; i += kProcThreads) {
      const int t = rows::token_at(list, i, wide);
      if (t >= a.vocab) {
        if (part == 0) atomicOr(a.status, CNNUE_STATUS_BAD_INDEX);
        continue;
      }
      const int s = t - lo;
      if (t < 0 || s < 0 || s >= width) continue;
      if (i < prompt)
        atomicOr(count + s, kSeen);
      else
        atomicAdd(count + s, 1u);
    }
  }
  if (BIAS) {
    btok = a.r.bias_tokens + row * a.r.bias_tokens_stride;
    bval = a.r.bias_values + row * a.r.bias_values_stride;
    for (int64_t k = threadIdx.x; k < a.r.bias_count; k += kProcThreads) {
      const int t = __ldg(btok + k);
      if (t >= a.vocab) {
        if (part == 0) atomicOr(a.status, CNNUE_STATUS_BAD_INDEX);
        continue;
      }
      const int s = t - lo;
      if (t >= 0 && s >= 0 && s < width) atomicMin(first + s, (uint32_t)k);
    }
    __syncthreads();
    for (int64_t k = threadIdx.x; k < a.r.bias_count; k += kProcThreads) {
      const int t = __ldg(btok + k);
      const int s = t - lo;
      if (t < 0 || t >= a.vocab || s < 0 || s >= width) continue;
      if ((first[s] & ~kRepeated) != (uint32_t)k) atomicOr(first + s, kRepeated);
    }
  }
  if (HIST || BIAS) __syncthreads();

  const bool whole = rows::lines_up(out, shift);
  const int v1 = v0 + a.vps;
  for (int v = v0 + threadIdx.x; v < v1; v += kProcThreads) {
    const int e0 = v * VE - shift;
    const uint32_t inside = rows::inside<VE>(e0, a.vocab);
    if (inside == 0) continue;
    const uint32_t ok = dead ? 0 : mask ? rows::allowed<VE>(mask, e0, a.vocab) : inside;
    float x[VE];
    rows::load(in, e0, inside, ok, kNegInf, x);
    if (HIST || BIAS) {
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        if (!(ok >> i & 1)) continue;
        if (HIST) {
          const uint32_t c = count[e0 + i - lo];
          if (c) {
            x[i] = x[i] > 0.f ? __fdiv_rn(x[i], rep) : __fmul_rn(x[i], rep);
            const uint32_t n = c & ~kSeen;
            if (n) x[i] = __fsub_rn(__fsub_rn(x[i], __fmul_rn(freq, (float)n)), pres);
          }
        }
        if (BIAS) {
          const uint32_t f = first[e0 + i - lo];
          if (f != kNoBias) {
            if (!(f & kRepeated)) {
              x[i] = __fadd_rn(x[i], __ldg(bval + f));
            } else {  // rare: walk the list from the first entry on
              for (int64_t k = f & ~kRepeated; k < a.r.bias_count; ++k)
                if (__ldg(btok + k) == e0 + i) x[i] = __fadd_rn(x[i], __ldg(bval + k));
            }
          }
        }
      }
    }
    rows::store<TO, VE>(out, e0, inside, whole, x);
  }
}

template <typename TI, typename TO, bool HIST, bool BIAS>
int launch_process(ProcArgs& a, int64_t n_rows, cudaStream_t s) {
  constexpr int VE = Vec<TI>::VE;
  const int64_t nv = rows::max_vectors<TI>(a.vocab);
  // 8192 tokens per slice: 32 KB of counters and 32 KB of bias slots at most
  const int64_t vps = std::min<int64_t>(nv, 8192 / VE);
  a.vps = (int)vps;
  a.split = (int)((nv + vps - 1) / vps);
  const size_t smem = (size_t)vps * VE * 4 * ((HIST ? 1 : 0) + (BIAS ? 1 : 0));
  if (n_rows * a.split > 0x7fffffff) return set_error(CNNUE_ERR_INVALID_ARG, "too many rows for one call");
  if (smem > 48 * 1024)
    CNNUE_CUDA_TRY(cudaFuncSetAttribute(process_kernel<TI, TO, HIST, BIAS>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  process_kernel<TI, TO, HIST, BIAS><<<(unsigned)(n_rows * a.split), kProcThreads, smem, s>>>(a);
  return check_launch_error("process_kernel");
}

template <typename TI, typename TO>
int pick_process(ProcArgs& a, int64_t n_rows, cudaStream_t s) {
  const bool hist = a.r.history && a.r.history_len > 0 && (a.r.repetition || a.r.frequency || a.r.presence);
  const bool bias = a.r.bias_tokens && a.r.bias_count > 0;
  if (hist) return bias ? launch_process<TI, TO, true, true>(a, n_rows, s) : launch_process<TI, TO, true, false>(a, n_rows, s);
  return bias ? launch_process<TI, TO, false, true>(a, n_rows, s) : launch_process<TI, TO, false, false>(a, n_rows, s);
}

// ---------------------------------------------------------------------------
// Masked softmax cross entropy.
//
//   A = allowed tokens, M = max_A z, S = sum_A exp(z - M), T = sum_A t,
//   D = sum_A t (M - z)
//   loss = w (T log S + D),   dloss/dz = w (T exp(z - M) / S - t) on A, 0 off it
//
// D and T log S instead of T lse - sum t z: a common offset of the logits
// does not cancel.
// ---------------------------------------------------------------------------

constexpr int kLossThreads = 256;

struct LossArgs {
  const void* z;
  int64_t z_stride;
  int vocab;
  cnnue_loss_targets t;
  const float* upstream;  // [rows] or null (backward pass)
  float* loss;            // [rows] or null
  float* stats;           // [rows][3]: M, S, T (written by the forward pass, read by the backward pass)
  void* grad;
  int64_t grad_stride;
  uint32_t* status;
};

template <typename T>
__device__ __forceinline__ float target_at(const void* p, int64_t i) {
  return Vec<T>::up(((const T*)p)[i]);
}
__device__ __forceinline__ float dense_target(const cnnue_loss_targets& t, int64_t i) {
  return t.dense_type == CNNUE_F32    ? target_at<float>(t.dense, i)
         : t.dense_type == CNNUE_BF16 ? target_at<__nv_bfloat16>(t.dense, i)
                                      : target_at<__half>(t.dense, i);
}

struct RowMask {
  const uint32_t* words;  // null: everything is allowed (unless dead)
  bool dead;
};
__device__ __forceinline__ RowMask row_mask(const cnnue_loss_targets& t, int64_t row, uint32_t* status, bool tell) {
  RowMask m{nullptr, false};
  if (!t.mask) return m;
  const int64_t i = t.mask_index ? (int64_t)t.mask_index[row] : t.mask_rows == 1 ? 0 : row;
  if (i >= t.mask_rows) {
    m.dead = true;
    if (tell) atomicOr(status, CNNUE_STATUS_BAD_INDEX);
  } else if (i >= 0) {
    m.words = t.mask + i * t.mask_stride;
  }
  return m;
}
__device__ __forceinline__ bool token_ok(const RowMask& m, int t) {
  return !m.dead && (!m.words || (__ldg(m.words + (t >> 5)) >> (t & 31) & 1));
}

struct Sums {
  float m, s, t, d;  // running maximum, sum of exp(z - m), target mass, sum of t (m - z)
};
// a += b, both relative to their own maxima.
__device__ __forceinline__ void join(Sums& a, const Sums& b) {
  const float m = rows::max_nan(a.m, b.m);
  if (m == kNegInf) {
    a.t += b.t;
    return;
  }
  const float fa = a.m == m ? 1.f : exp2f((a.m - m) * rows::kLog2e), fb = b.m == m ? 1.f : exp2f((b.m - m) * rows::kLog2e);
  // a side without allowed logits above -inf has s = 0; its mass sits on -inf logits
  a.d = (a.t != 0.f ? a.d + a.t * (m - a.m) : 0.f) + (b.t != 0.f ? b.d + b.t * (m - b.m) : 0.f);
  a.s = a.s * fa + b.s * fb;
  a.t += b.t;
  a.m = m;
}

__device__ __forceinline__ Sums block_join(Sums v, Sums* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Sums u;
    u.m = __shfl_xor_sync(~0u, v.m, o);
    u.s = __shfl_xor_sync(~0u, v.s, o);
    u.t = __shfl_xor_sync(~0u, v.t, o);
    u.d = __shfl_xor_sync(~0u, v.d, o);
    // both lanes of a pair form the same sum in the same order
    if (threadIdx.x & o) {
      join(u, v);
      v = u;
    } else {
      join(v, u);
    }
  }
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < kLossThreads / 32; ++w) join(v, shared[w]);
  return v;
}

// One CTA per row.  FWD: the row's sums, loss and stats.  GRAD: the gradient
// (with !FWD from the stats of an earlier forward pass).
template <typename T, bool FWD, bool GRAD>
__global__ void __launch_bounds__(kLossThreads) loss_kernel(const LossArgs a) {
  constexpr int VE = Vec<T>::VE;
  __shared__ Sums shared[kLossThreads / 32];
  const int64_t row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.z_stride;
  const int shift = rows::shift_of(z);
  const int nv = (shift + a.vocab + VE - 1) / VE;
  const bool wide = a.t.index_bytes == 8;
  const char* list = a.t.index ? (const char*)a.t.index + row * a.t.index_stride * a.t.index_bytes : nullptr;
  const float* prob = a.t.prob ? a.t.prob + row * a.t.prob_stride : nullptr;
  float w = a.t.weights ? a.t.weights[row] : 1.f;
  const bool idle = w == 0.f;  // a padded row: not read, loss and gradient 0
  const RowMask mask = row_mask(a.t, row, a.status, threadIdx.x == 0);

  Sums v{kNegInf, 0.f, 0.f, 0.f};
  if (FWD && !idle) {
    for (int i = threadIdx.x; i < nv; i += kLossThreads) {
      const int e0 = i * VE - shift;
      const uint32_t in = rows::inside<VE>(e0, a.vocab);
      const uint32_t ok = mask.dead ? 0 : mask.words ? rows::allowed<VE>(mask.words, e0, a.vocab) : in;
      if (ok == 0) continue;
      float x[VE];
      rows::load(z, e0, in, ok, kNegInf, x);
      Sums u{x[0], 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 1; j < VE; ++j) u.m = rows::max_nan(u.m, x[j]);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        if (u.m != kNegInf) u.s += exp2f((x[j] - u.m) * rows::kLog2e);
        if (a.t.dense && (ok >> j & 1)) {
          const float t = dense_target(a.t, row * a.t.dense_stride + e0 + j);
          if (t != 0.f) {
            u.t += t;
            if (u.m != kNegInf) u.d += t * (u.m - x[j]);
          }
        }
      }
      join(v, u);
    }
    v = block_join(v, shared);
    if (list) {  // every thread forms the same sums in list order
      for (int64_t k = 0; k < a.t.count; ++k) {
        const int tok = rows::token_at(list, k, wide);
        if (tok >= a.vocab) {
          if (threadIdx.x == 0) atomicOr(a.status, CNNUE_STATUS_BAD_INDEX);
          continue;
        }
        const float t = tok < 0 || !token_ok(mask, tok) ? 0.f : prob ? prob[k] : 1.f;
        if (t != 0.f) {
          v.t += t;
          v.d += t * (v.m - Vec<T>::up(z[tok]));
        }
      }
    }
    if (threadIdx.x == 0) {
      if (a.loss) a.loss[row] = v.m == kNegInf ? 0.f : w * ((v.t != 0.f ? v.t * logf(v.s) : 0.f) + v.d);
      if (a.stats) {
        a.stats[3 * row] = v.m;
        a.stats[3 * row + 1] = v.s;
        a.stats[3 * row + 2] = v.t;
      }
    }
  } else if (FWD && threadIdx.x == 0) {
    if (a.loss) a.loss[row] = 0.f;
    if (a.stats) a.stats[3 * row] = kNegInf;
  }
  if (!GRAD) return;
  if (!FWD) v.m = a.stats[3 * row], v.s = a.stats[3 * row + 1], v.t = a.stats[3 * row + 2];
  if (a.upstream) w *= a.upstream[row];
  T* g = (T*)a.grad + row * a.grad_stride;
  const bool whole = rows::lines_up(g, shift);
  const bool none = idle || v.m == kNegInf;  // nothing is left of the row
  const float c = none || v.t == 0.f ? 0.f : w * v.t / v.s;
  for (int i = threadIdx.x; i < nv; i += kLossThreads) {
    const int e0 = i * VE - shift;
    const uint32_t in = rows::inside<VE>(e0, a.vocab);
    const uint32_t ok = none || mask.dead ? 0 : mask.words ? rows::allowed<VE>(mask.words, e0, a.vocab) : in;
    float x[VE];
    rows::load(z, e0, in, c == 0.f ? 0 : ok, kNegInf, x);
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float t = a.t.dense && (ok >> j & 1) ? dense_target(a.t, row * a.t.dense_stride + e0 + j) : 0.f;
      x[j] = ok >> j & 1 ? (c == 0.f ? 0.f : c * exp2f((x[j] - v.m) * rows::kLog2e)) - w * t : 0.f;
    }
    rows::store<T, VE>(g, e0, in, whole, x);
  }
  if (!list || none) return;
  __syncthreads();  // the listed tokens' elements again, now with their targets
  for (int64_t k = threadIdx.x; k < a.t.count; k += kLossThreads) {
    const int tok = rows::token_at(list, k, wide);
    if (tok < 0 || tok >= a.vocab || !token_ok(mask, tok)) continue;
    float t = 0.f;
    bool again = false;  // a token named before belongs to its first entry
    for (int64_t j = 0; j < a.t.count; ++j) {
      if (rows::token_at(list, j, wide) != tok) continue;
      if (j < k) {
        again = true;
        break;
      }
      t += prob ? prob[j] : 1.f;
    }
    if (again) continue;
    g[tok] = Vec<T>::down((c == 0.f ? 0.f : c * exp2f((Vec<T>::up(z[tok]) - v.m) * rows::kLog2e)) - w * t);
  }
}

template <typename T, bool FWD, bool GRAD>
int launch_loss(const LossArgs& a, int64_t n_rows, cudaStream_t s) {
  if (n_rows > 0x7fffffff) return set_error(CNNUE_ERR_INVALID_ARG, "too many rows for one call");
  loss_kernel<T, FWD, GRAD><<<(unsigned)n_rows, kLossThreads, 0, s>>>(a);
  return check_launch_error("loss_kernel");
}

template <bool FWD, bool GRAD>
int pick_loss(const LossArgs& a, int type, int64_t n_rows, cudaStream_t s) {
  if (type == CNNUE_F32) return launch_loss<float, FWD, GRAD>(a, n_rows, s);
  if (type == CNNUE_BF16) return launch_loss<__nv_bfloat16, FWD, GRAD>(a, n_rows, s);
  return launch_loss<__half, FWD, GRAD>(a, n_rows, s);
}

// ---- argument checks --------------------------------------------------------
int element_bytes(int type) { return type == CNNUE_F32 ? 4 : type == CNNUE_BF16 || type == CNNUE_F16 ? 2 : 0; }

int check_rows(const void* p, int64_t stride, int type, int64_t n_rows, int64_t vocab, bool written, const char* what) {
  const int b = element_bytes(type);
  if (!b) return set_error(CNNUE_ERR_INVALID_ARG, "%s: unknown element type %d", what, type);
  if (!p) return set_error(CNNUE_ERR_INVALID_ARG, "%s: null buffer", what);
  if ((uintptr_t)p % b) return set_error(CNNUE_ERR_INVALID_ARG, "%s: not aligned to its elements", what);
  if (stride < 0 || (written && n_rows > 1 && stride < vocab))
    return set_error(CNNUE_ERR_INVALID_ARG, "%s: row stride %lld", what, (long long)stride);
  return CNNUE_OK;
}

int check_mask(const uint32_t* mask, int64_t stride, int64_t mask_rows, const int32_t* index, int64_t n_rows, int64_t vocab) {
  if (!mask) return index ? set_error(CNNUE_ERR_INVALID_ARG, "mask_index without a mask") : CNNUE_OK;
  if (mask_rows < 0 || stride < 0 || (mask_rows > 1 && stride < (vocab + 31) / 32))
    return set_error(CNNUE_ERR_INVALID_ARG, "mask: rows or stride");
  if (!index && mask_rows != 1 && mask_rows != n_rows)
    return set_error(CNNUE_ERR_INVALID_ARG, "mask: %lld rows for %lld rows of logits", (long long)mask_rows,
                     (long long)n_rows);
  return CNNUE_OK;
}

// Whether [p, ...) and [q, ...) of the two row sets share a byte.
bool overlap(const void* p, int64_t p_stride, int pb, const void* q, int64_t q_stride, int qb, int64_t n_rows,
             int64_t vocab) {
  const uintptr_t p0 = (uintptr_t)p, p1 = p0 + ((n_rows - 1) * p_stride + vocab) * pb;
  const uintptr_t q0 = (uintptr_t)q, q1 = q0 + ((n_rows - 1) * q_stride + vocab) * qb;
  return p0 < q1 && q0 < p1;
}

int check_targets(const cnnue_loss_targets* t, int64_t n_rows, int64_t vocab) {
  if (!t) return set_error(CNNUE_ERR_INVALID_ARG, "null targets");
  if ((t->dense != nullptr) == (t->index != nullptr))
    return set_error(CNNUE_ERR_INVALID_ARG, "targets: give either dense targets or a list");
  if (t->dense) {
    if (int st = check_rows(t->dense, t->dense_stride, t->dense_type, n_rows, vocab, false, "targets")) return st;
    if (t->prob) return set_error(CNNUE_ERR_INVALID_ARG, "targets: probabilities without a list");
  } else {
    if (t->index_bytes != 4 && t->index_bytes != 8) return set_error(CNNUE_ERR_INVALID_ARG, "targets: index_bytes");
    if (t->count < 0 || t->index_stride < 0 || t->prob_stride < 0)
      return set_error(CNNUE_ERR_INVALID_ARG, "targets: negative size");
  }
  return check_mask(t->mask, t->mask_stride, t->mask_rows, t->mask_index, n_rows, vocab);
}

int check_shape(int64_t n_rows, int64_t vocab, const uint32_t* status) {
  if (n_rows < 0 || vocab < 0 || vocab > kMaxVocab) return set_error(CNNUE_ERR_INVALID_ARG, "rows or vocabulary size");
  if (!status) return set_error(CNNUE_ERR_INVALID_ARG, "null status word");
  return CNNUE_OK;
}

}  // namespace
}  // namespace logits
}  // namespace cnnue

using namespace cnnue;
using namespace cnnue::logits;

extern "C" {

int cnnue_logits_process(const void* d_logits, int64_t logits_stride, int logits_type, void* d_out, int64_t out_stride,
                         int out_type, int64_t n_rows, int64_t vocab, const cnnue_logit_rules* rules,
                         uint32_t* d_status, void* stream) {
  if (int st = check_shape(n_rows, vocab, d_status)) return st;
  if (!rules) return set_error(CNNUE_ERR_INVALID_ARG, "null rules");
  if (n_rows == 0 || vocab == 0) return CNNUE_OK;
  if (int st = check_rows(d_logits, logits_stride, logits_type, n_rows, vocab, false, "logits")) return st;
  if (int st = check_rows(d_out, out_stride, out_type, n_rows, vocab, true, "out")) return st;
  if (out_type != logits_type && out_type != CNNUE_F32)
    return set_error(CNNUE_ERR_INVALID_ARG, "out has the logits' type or fp32");
  const bool in_place = d_logits == d_out && out_type == logits_type && (logits_stride == out_stride || n_rows == 1);
  if (!in_place && overlap(d_logits, logits_stride, element_bytes(logits_type), d_out, out_stride,
                           element_bytes(out_type), n_rows, vocab))
    return set_error(CNNUE_ERR_INVALID_ARG, "out overlaps the logits without being the same rows");
  const cnnue_logit_rules& r = *rules;
  if (r.history) {
    if (r.history_bytes != 4 && r.history_bytes != 8) return set_error(CNNUE_ERR_INVALID_ARG, "history_bytes");
    if (r.history_len < 0 || r.history_len >= kSeen || r.history_stride < 0)
      return set_error(CNNUE_ERR_INVALID_ARG, "history: length or stride");
  } else if (r.repetition || r.frequency || r.presence || r.lengths || r.prompt_lengths) {
    return set_error(CNNUE_ERR_INVALID_ARG, "penalties without a history");
  }
  if ((r.bias_tokens != nullptr) != (r.bias_values != nullptr))
    return set_error(CNNUE_ERR_INVALID_ARG, "bias tokens and values come together");
  if (r.bias_count < 0 || r.bias_count >= kNoBias || r.bias_tokens_stride < 0 || r.bias_values_stride < 0)
    return set_error(CNNUE_ERR_INVALID_ARG, "bias: count or stride");
  if (int st = check_mask(r.mask, r.mask_stride, r.mask_rows, r.mask_index, n_rows, vocab)) return st;
  ProcArgs a{d_logits, d_out, logits_stride, out_stride, (int)vocab, 0, 0, r, d_status};
  cudaStream_t s = (cudaStream_t)stream;
  if (logits_type == CNNUE_F32) return pick_process<float, float>(a, n_rows, s);
  if (logits_type == CNNUE_BF16)
    return out_type == CNNUE_F32 ? pick_process<__nv_bfloat16, float>(a, n_rows, s)
                                 : pick_process<__nv_bfloat16, __nv_bfloat16>(a, n_rows, s);
  return out_type == CNNUE_F32 ? pick_process<__half, float>(a, n_rows, s) : pick_process<__half, __half>(a, n_rows, s);
}

int cnnue_policy_loss_fwd(const void* d_logits, int64_t logits_stride, int logits_type, int64_t n_rows, int64_t vocab,
                          const cnnue_loss_targets* targets, float* d_loss, float* d_stats, uint32_t* d_status,
                          void* stream) {
  if (int st = check_shape(n_rows, vocab, d_status)) return st;
  if (n_rows == 0) return CNNUE_OK;
  if (int st = check_targets(targets, n_rows, vocab)) return st;
  if (vocab == 0) return set_error(CNNUE_ERR_INVALID_ARG, "empty vocabulary");
  if (int st = check_rows(d_logits, logits_stride, logits_type, n_rows, vocab, false, "logits")) return st;
  if (!d_loss || !d_stats) return set_error(CNNUE_ERR_INVALID_ARG, "null loss or stats");
  const LossArgs a{d_logits, logits_stride, (int)vocab, *targets, nullptr, d_loss, d_stats, nullptr, 0, d_status};
  return pick_loss<true, false>(a, logits_type, n_rows, (cudaStream_t)stream);
}

int cnnue_policy_loss_bwd(const void* d_logits, int64_t logits_stride, int logits_type, int64_t n_rows, int64_t vocab,
                          const cnnue_loss_targets* targets, const float* d_stats, const float* d_upstream, void* d_grad,
                          int64_t grad_stride, uint32_t* d_status, void* stream) {
  if (int st = check_shape(n_rows, vocab, d_status)) return st;
  if (n_rows == 0) return CNNUE_OK;
  if (int st = check_targets(targets, n_rows, vocab)) return st;
  if (vocab == 0) return set_error(CNNUE_ERR_INVALID_ARG, "empty vocabulary");
  if (int st = check_rows(d_logits, logits_stride, logits_type, n_rows, vocab, false, "logits")) return st;
  if (int st = check_rows(d_grad, grad_stride, logits_type, n_rows, vocab, true, "grad")) return st;
  if (!d_stats) return set_error(CNNUE_ERR_INVALID_ARG, "null stats");
  const int b = element_bytes(logits_type);
  if (overlap(d_logits, logits_stride, b, d_grad, grad_stride, b, n_rows, vocab))
    return set_error(CNNUE_ERR_INVALID_ARG, "grad overlaps the logits");
  const LossArgs a{d_logits,   logits_stride, (int)vocab, *targets,    d_upstream, nullptr, const_cast<float*>(d_stats),
                   d_grad, grad_stride, d_status};
  return pick_loss<false, true>(a, logits_type, n_rows, (cudaStream_t)stream);
}

int cnnue_policy_loss_grad(const void* d_logits, int64_t logits_stride, int logits_type, int64_t n_rows, int64_t vocab,
                           const cnnue_loss_targets* targets, float* d_loss, void* d_grad, int64_t grad_stride,
                           uint32_t* d_status, void* stream) {
  if (int st = check_shape(n_rows, vocab, d_status)) return st;
  if (n_rows == 0) return CNNUE_OK;
  if (int st = check_targets(targets, n_rows, vocab)) return st;
  if (vocab == 0) return set_error(CNNUE_ERR_INVALID_ARG, "empty vocabulary");
  if (int st = check_rows(d_logits, logits_stride, logits_type, n_rows, vocab, false, "logits")) return st;
  if (int st = check_rows(d_grad, grad_stride, logits_type, n_rows, vocab, true, "grad")) return st;
  if (!d_loss) return set_error(CNNUE_ERR_INVALID_ARG, "null loss");
  const int b = element_bytes(logits_type);
  if (overlap(d_logits, logits_stride, b, d_grad, grad_stride, b, n_rows, vocab))
    return set_error(CNNUE_ERR_INVALID_ARG, "grad overlaps the logits");
  const LossArgs a{d_logits, logits_stride, (int)vocab, *targets, nullptr, d_loss, nullptr, d_grad, grad_stride, d_status};
  return pick_loss<true, true>(a, logits_type, n_rows, (cudaStream_t)stream);
}

}  // extern "C"
