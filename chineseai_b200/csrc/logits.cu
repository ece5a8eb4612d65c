// logits.cu - what a model may answer with, and what it learns from: penalties,
// biases and masks on rows of logits, and the masked softmax cross entropy
// with its gradient.  Rows are [vocab] of fp32, bf16 or fp16 at any stride;
// arithmetic is fp32, rounded once at the store.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "rowvec.cuh"

namespace cnnue {
namespace logits {
namespace {

namespace cg = cooperative_groups;
using rows::kNegInf;
using rows::Vec;

constexpr int64_t kMaxVocab = (int64_t)1 << 30;  // element offsets inside a row are 32-bit

// ---------------------------------------------------------------------------
// What both operators share: a row's mask, a CTA's slice of a row, and the
// tokens that a list may name more than once.
// ---------------------------------------------------------------------------

struct RowMask {
  const uint32_t* words;  // null: everything is allowed (unless dead)
  bool dead;
};
template <typename Rules>  // cnnue_logit_rules or cnnue_loss_targets
__device__ __forceinline__ RowMask row_mask(const Rules& t, int64_t row, uint32_t* status, bool tell) {
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

// A CTA's slice of a row: vectors 0 .. n - 1, vector i at element first + i VE.
// All but the row's first and last are whole; whole ones are [from, to).
template <int VE>
struct Slice {
  int first, n, from, to, lo, hi;
  __device__ __forceinline__ Slice(int rank, int vps, int shift, int vocab) {
    first = rank * vps * VE - shift;
    n = max(0, min(vps, (shift + vocab + VE - 1) / VE - rank * vps));
    from = n > 0 && first < 0 ? 1 : 0;
    to = n > 0 && first + n * VE > vocab ? n - 1 : n;
    lo = max(0, first);
    hi = min(vocab, first + n * VE);
  }
  // f(i, e0, n) for this thread's share of the whole vectors, n = N (the
  // vectors i + j blockDim, at e0 + j blockDim VE) and 1 for what is left.  The
  // same share at every call.
  template <int N, typename F>
  __device__ __forceinline__ void each(F&& f) const {
    const int stride = blockDim.x;
    int i = from + threadIdx.x;
    for (; i + (N - 1) * stride < to; i += N * stride) f(i, first + i * VE, std::integral_constant<int, N>{});
    if (N > 1) {
#pragma unroll 1
      for (; i < to; i += stride) f(i, first + i * VE, std::integral_constant<int, 1>{});
    }
  }
  // f(first element) for the partial vectors, by two threads.
  template <typename F>
  __device__ __forceinline__ void edges(F&& f) const {
    if (threadIdx.x == 0 && from == 1) f(first);
    if (threadIdx.x == blockDim.x - 1 && to < n && (n > 1 || from == 0)) f(first + (n - 1) * VE);
  }
};

// Which of a list's tokens may occur in it more than once: a token's bit (by
// its low 13 bits) is set a second time.  Tokens that share a bit by chance
// are marked too, which costs time, not results.
struct Repeats {
  static constexpr int kWords = 256;
  uint32_t once[kWords], more[kWords];
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kWords; i += blockDim.x) once[i] = more[i] = 0;
  }
  __device__ __forceinline__ void mark(int tok) {
    const uint32_t word = (uint32_t)tok / 32 % kWords, bit = 1u << (tok & 31);
    if (atomicOr(once + word, bit) & bit) atomicOr(more + word, bit);
  }
  __device__ __forceinline__ bool marked(int tok) const { return more[(uint32_t)tok / 32 % kWords] >> (tok & 31) & 1; }
};

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
// Every step is one IEEE fp32 operation.  Two parts: the rows are streamed
// through the mask (what that excludes is not read), and the tokens that are
// penalised or biased, a few hundred or thousand of a row, are computed from
// their logits, which are in L2 by then, and stored over.  The second part
// needs to know how often a token occurs: shared memory counts it, by integer
// atomics (their order does not change the counts), and the occurrence that
// found the counter at 0 computes the token.
//
// A row of up to kFusedTokens tokens is one CTA's, both parts in one launch.
// Longer rows are streamed by as many CTAs as they need and the second part is
// a launch of its own, whose reading and counting overlap the streaming
// (programmatic dependent launch).  With the counting in every slice's CTA
// instead, each read the whole history and had few threads left to stream:
// 135 us for 2048 x 50001 fp16 with 512 tokens of history, 37 us for 64 x
// 131072 bf16 with 8192; now 97 us (streaming alone 67) and 24.
// ---------------------------------------------------------------------------

constexpr int kProcThreads = 256;
constexpr int kProcAhead = 4;        // vectors per thread in flight
constexpr int kFusedTokens = 16384;  // 32 or 64 KB of counters
constexpr int kCountThreads = 512;
constexpr int kTokensAhead = 4;  // history tokens per thread that are read first of all,
constexpr int kMoreTokens = 8;   // and after those, in flight
constexpr int64_t kMostTokens = 0x7fff0000;  // longest history (its positions plus a round of a CTA fit 31 bits)
constexpr int kCountBytes = 144 * 1024;  // the largest Table
constexpr int kHashTokens = kCountThreads * kTokensAhead;  // the longest history that is counted in a hash table

struct ProcArgs {
  const void* in;
  void* out;
  int64_t in_stride, out_stride;
  int vocab, split, vps;  // streaming: slices per row, vectors per slice
  int slots, lg;          // counting: counters per CTA; 1 << lg CTAs per row
  bool in_place;
  cnnue_logit_rules r;
  uint32_t* status;
};

// Streams one slice of a row through the mask.
template <typename TI, typename TO>
__device__ __forceinline__ void stream_slice(const ProcArgs& a, const TI* in, TO* out, int part, const RowMask& mask) {
  constexpr int VE = Vec<TI>::VE;
  const int shift = rows::shift_of(in), stride = blockDim.x;
  const Slice<VE> slice(part, a.vps, shift, a.vocab);
  const bool lines_up = rows::lines_up(out, shift);
  slice.template each<kProcAhead>([&](int, int e0, auto n) {
    constexpr int N = decltype(n)::value;
    uint4 raw[N];
    uint32_t ok[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = e0 + j * stride * VE;
      ok[j] = mask.dead ? 0 : mask.words ? rows::allowed_whole<VE>(mask.words, e) : rows::kFull<VE>;
      raw[j] = make_uint4(0, 0, 0, 0);
      if (ok[j] && !(a.in_place && ok[j] == rows::kFull<VE>)) raw[j] = rows::load16(in + e);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (a.in_place && ok[j] == rows::kFull<VE>) continue;  // nothing changes
      const int e = e0 + j * stride * VE;
      if (ok[j] != rows::kFull<VE>) raw[j] = Vec<TI>::only(raw[j], ok[j]);
      if (sizeof(TI) == sizeof(TO) && lines_up) {
        *reinterpret_cast<uint4*>(out + e) = raw[j];
      } else {
        float x[VE];
        Vec<TI>::unpack(raw[j], x);
        rows::store<TO, VE>(out, e, rows::kFull<VE>, lines_up, x);
      }
    }
  });
  slice.edges([&](int e0) {
    const uint32_t in_row = rows::inside<VE>(e0, a.vocab);
    const uint32_t ok = mask.dead ? 0 : mask.words ? rows::allowed<VE>(mask.words, e0, a.vocab) : in_row;
    float x[VE];
    Vec<TI>::unpack(Vec<TI>::only(rows::load_raw(in, e0, in_row, ok), ok), x);
    rows::store<TO, VE>(out, e0, in_row, false, x);
  });
}

// What a CTA knows of its tokens, in shared memory: a slot per token, with a
// counter of BITS bits (the high bit says that the token occurs, the others
// how often after the prompt; 16 bits do for histories of up to 32767 tokens),
// two bits for the bias list (named once, named again), and a list of slots.
// HASH: the slots are a hash table of tokens, at most half full, for short
// histories over any vocabulary; else CTA p of the row's 1 << lg owns the tokens
// t with t mod (1 << lg) = p, token t in slot t >> lg (text uses low tokens
// most: neighbours are dealt to different CTAs).
template <int BITS, bool HASH>
struct Table {
  static constexpr uint32_t kSeen = 1u << (BITS - 1);
  uint32_t *words, *keys, *once, *more;
  uint16_t* list;
  int* listed;
  int slots, lg;

  static __host__ __device__ size_t bytes(int64_t slots, bool bias, int64_t longest) {
    return (size_t)((slots * BITS / 8 + 15) / 16 * 16 + (HASH ? slots * 4 : 0) + (bias ? (slots + 31) / 32 * 8 : 0) +
                    (HASH ? 0 : 2 * (slots < longest ? slots : longest)) + 16);
  }
  __device__ __forceinline__ Table(void* smem, int* counter, int n, int log_ctas, bool bias)
      : listed(counter), slots(n), lg(log_ctas) {
    words = (uint32_t*)smem;
    keys = words + (slots * BITS / 8 + 15) / 16 * 4;
    once = keys + (HASH ? slots : 0);
    more = once + (bias ? (slots + 31) / 32 : 0);
    list = (uint16_t*)(more + (bias ? (slots + 31) / 32 : 0));
  }
  __device__ __forceinline__ void clear(bool bias) const {
    for (int i = threadIdx.x; i < (slots * BITS / 8 + 15) / 16; i += blockDim.x)
      reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
    if (HASH)
      for (int i = threadIdx.x; i < slots; i += blockDim.x) keys[i] = ~0u;
    if (bias)
      for (int i = threadIdx.x; i < (slots + 31) / 32; i += blockDim.x) once[i] = more[i] = 0;
    if (threadIdx.x == 0) *listed = 0;
  }
  // The slot of token t (the table holds it, or gets it).
  __device__ __forceinline__ int slot(int t) const {
    if (!HASH) return t >> lg;
    uint32_t h = (uint32_t)t * 2654435761u >> __clz(slots - 1);
    for (int n = 0; n < slots; ++n) {  // ends at a free slot: half of them are
      const uint32_t k = atomicCAS(keys + h, ~0u, (uint32_t)t);
      if (k == ~0u || k == (uint32_t)t) break;
      h = (h + 1) & (slots - 1);
    }
    return (int)h;
  }
  __device__ __forceinline__ int token(int s, int part) const { return s << lg | part; }
  // Counts the tokens in slots s[0..N) (negative: none) at positions i, i +
  // stride, ..; bit j of the result: s[j] had not occurred.
  template <int N>
  __device__ __forceinline__ uint32_t see(const int* s, int i, int stride, int prompt) const {
    uint32_t before[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int at = BITS == 16 ? 16 * (s[j] & 1) : 0;
      uint32_t* w = words + (BITS == 16 ? s[j] >> 1 : s[j]);
      const bool said = i + j * stride >= prompt;
      before[j] = ~0u;
      if (s[j] >= 0 && said) before[j] = atomicAdd(w, 1u << at);
      if (s[j] >= 0 && !said) before[j] = atomicOr(w, kSeen << at);
    }
    uint32_t first = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (s[j] >= 0 && (BITS == 16 ? before[j] >> 16 * (s[j] & 1) & 0xffffu : before[j]) == 0) first |= 1u << j;
    return first;
  }
  // The slots s[j] that `which` names to the list; called by whole warps.
  template <int N>
  __device__ __forceinline__ void note(const int* s, uint32_t which) const {
    const int lane = threadIdx.x & 31, n = __popc(which);
    int at = n;  // inclusive sums over the warp
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(~0u, at, o);
      if (lane >= o) at += v;
    }
    int base = 0;
    if (lane == 31 && at > 0) base = atomicAdd(listed, at);
    at += __shfl_sync(~0u, base, 31) - n;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (which >> j & 1) list[at++] = (uint16_t)s[j];
  }
  __device__ __forceinline__ uint32_t count(int s) const {
    return BITS == 16 ? words[s >> 1] >> 16 * (s & 1) & 0xffffu : words[s];
  }
  __device__ __forceinline__ void mark(int s) const {
    const uint32_t bit = 1u << (s & 31);
    if (atomicOr(once + (s >> 5), bit) & bit) atomicOr(more + (s >> 5), bit);
  }
  __device__ __forceinline__ bool biased(int s) const { return once[s >> 5] >> (s & 31) & 1; }
  __device__ __forceinline__ bool again(int s) const { return more[s >> 5] >> (s & 31) & 1; }
};

struct Penalties {
  float rep = 1.f, freq = 0.f, pres = 0.f;
  // `c`: a counter, 0 = the token does not occur.
  template <int BITS>
  __device__ __forceinline__ float apply(float x, uint32_t c) const {
    if (c == 0) return x;
    x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    const uint32_t n = c & ~(1u << (BITS - 1));
    return n ? __fsub_rn(__fsub_rn(x, __fmul_rn(freq, (float)n)), pres) : x;
  }
};

// The penalised and biased tokens of a row that CTA `part` owns.  `streamed()`
// is called before the first store, when the loads that need not wait for the
// streamed row are under way.
template <typename TI, typename TO, int BITS, bool HASH, typename F>
__device__ __forceinline__ void penalise(const ProcArgs& a, const TI* in, TO* out, int64_t row, int part,
                                         const RowMask& mask, void* smem, F&& streamed) {
  __shared__ int listed;
  const int stride = blockDim.x;
  const bool hist = a.r.history != nullptr, bias = a.r.bias_tokens != nullptr;
  const Table<BITS, HASH> table(smem, &listed, a.slots, a.lg, bias);
  Penalties pen;
  const int most = hist ? (int)a.r.history_len : 0;  // below kMostTokens: positions are 32-bit
  int len = most, prompt = 0;
  const bool wide = a.r.history_bytes == 8;
  const char* list = (const char*)a.r.history + row * a.r.history_stride * a.r.history_bytes;
  int ahead[kTokensAhead];
#pragma unroll
  for (int j = 0; j < kTokensAhead; ++j) {
    const int i = threadIdx.x + j * stride;
    ahead[j] = i < most ? rows::token_at(list, i, wide) : -1;
  }
  if (hist) {
    if (a.r.lengths) len = a.r.lengths[row];
    if (a.r.prompt_lengths) prompt = a.r.prompt_lengths[row];
    if (a.r.repetition) pen.rep = a.r.repetition[row];
    if (a.r.frequency) pen.freq = a.r.frequency[row];
    if (a.r.presence) pen.pres = a.r.presence[row];
  }
  const int32_t* btok = a.r.bias_tokens + row * a.r.bias_tokens_stride;
  const float* bval = a.r.bias_values + row * a.r.bias_values_stride;
  int biased = bias && threadIdx.x < a.r.bias_count ? __ldg(btok + threadIdx.x) : -1;
  table.clear(bias);

  bool bad = false;
  auto own = [&](int t) {  // t, or -1 if it is none of this CTA's tokens
    bad |= t >= a.vocab;
    return t >= 0 && t < a.vocab && (HASH || (t & ((1 << a.lg) - 1)) == part) ? t : -1;
  };
  auto value = [&](int t) { return Vec<TI>::up(in[t]); };
  float x[kTokensAhead], x_biased = 0.f;
  uint32_t mine = 0, stays = 0;  // bit j: token j is this thread's to compute; the mask allows it
  if (len < 0 || len > most) {
    if (threadIdx.x == 0 && part == 0) atomicOr(a.status, CNNUE_STATUS_BAD_OFFSETS);
    len = max(0, min(len, most));
  }
#pragma unroll
  for (int j = 0; j < kTokensAhead; ++j) {
    ahead[j] = (int)threadIdx.x + j * stride < len ? own(ahead[j]) : -1;
    x[j] = ahead[j] >= 0 ? value(ahead[j]) : 0.f;
    if (ahead[j] >= 0 && token_ok(mask, ahead[j])) stays |= 1u << j;
  }
  biased = own(biased);
  if (biased >= 0 && !token_ok(mask, biased)) biased = -1;
  if (biased >= 0) x_biased = value(biased);
  __syncthreads();  // cleared

  int at[kTokensAhead], at_biased = -1;
#pragma unroll
  for (int j = 0; j < kTokensAhead; ++j) at[j] = ahead[j] >= 0 ? table.slot(ahead[j]) : -1;
  mine = table.template see<kTokensAhead>(at, threadIdx.x, stride, prompt);
  if (!HASH) {  // a hash table's histories end here
    for (int b = kTokensAhead * stride; b < len; b += kMoreTokens * stride) {  // the same for all threads
      const int i = b + threadIdx.x;
      int s[kMoreTokens];
#pragma unroll
      for (int j = 0; j < kMoreTokens; ++j) s[j] = i + j * stride < len ? rows::token_at(list, i + j * stride, wide) : -1;
#pragma unroll
      for (int j = 0; j < kMoreTokens; ++j) s[j] = own(s[j]) >= 0 ? table.slot(s[j]) : -1;
      const uint32_t first = table.template see<kMoreTokens>(s, i, stride, prompt);
      table.template note<kMoreTokens>(s, first);
    }
  }
  if (biased >= 0) table.mark(at_biased = table.slot(biased));
  if (bias) {
    for (int64_t k = threadIdx.x + stride; k < a.r.bias_count; k += stride) {
      const int t = own(__ldg(btok + k));
      if (t >= 0 && token_ok(mask, t)) table.mark(table.slot(t));
    }
  }
  if (bad && part == 0) atomicOr(a.status, CNNUE_STATUS_BAD_INDEX);
  __syncthreads();  // counted
  streamed();

#pragma unroll
  for (int j = 0; j < kTokensAhead; ++j)  // a biased token: below
    if ((mine & stays & 1u << j) && !(bias && table.biased(at[j])))
      out[ahead[j]] = Vec<TO>::down(pen.apply<BITS>(x[j], table.count(at[j])));
  if (!HASH) {
    const int n = listed;
    for (int i = threadIdx.x; i < n; i += kTokensAhead * stride) {
      int s[kTokensAhead], t[kTokensAhead];
#pragma unroll
      for (int j = 0; j < kTokensAhead; ++j) {
        s[j] = i + j * stride < n ? table.list[i + j * stride] : -1;
        if (s[j] < 0) continue;
        t[j] = table.token(s[j], part);
        x[j] = value(t[j]);
        if (!token_ok(mask, t[j]) || (bias && table.biased(s[j]))) s[j] = -1;
      }
#pragma unroll
      for (int j = 0; j < kTokensAhead; ++j)
        if (s[j] >= 0) out[t[j]] = Vec<TO>::down(pen.apply<BITS>(x[j], table.count(s[j])));
    }
  }
  auto add_bias = [&](int64_t k, int t, int s, float y) {
    y = pen.apply<BITS>(y, table.count(s));
    if (!table.again(s)) {
      y = __fadd_rn(y, __ldg(bval + k));
    } else {  // in list order, by the thread of the token's first entry
      bool earlier = false;
      for (int64_t j = 0; j < a.r.bias_count; ++j) {
        if (__ldg(btok + j) != t) continue;
        earlier |= j < k;
        y = __fadd_rn(y, __ldg(bval + j));
      }
      if (earlier) return;
    }
    out[t] = Vec<TO>::down(y);
  };
  if (biased >= 0) add_bias(threadIdx.x, biased, at_biased, x_biased);
  if (bias) {
    for (int64_t k = threadIdx.x + stride; k < a.r.bias_count; k += stride) {
      const int t = own(__ldg(btok + k));
      // in place, a later entry of a token finds it written, and leaves it: its slot is marked
      if (t >= 0 && token_ok(mask, t)) add_bias(k, t, table.slot(t), value(t));
    }
  }
}

template <typename TI, typename TO>
__global__ void __launch_bounds__(kProcThreads, 8) stream_kernel(const __grid_constant__ ProcArgs a) {
  const int64_t row = blockIdx.x / (unsigned)a.split;
  const int part = (int)(blockIdx.x % (unsigned)a.split);
  const RowMask mask = row_mask(a.r, row, a.status, threadIdx.x == 0 && part == 0);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  stream_slice<TI, TO>(a, (const TI*)a.in + row * a.in_stride, (TO*)a.out + row * a.out_stride, part, mask);
}

template <typename TI, typename TO, int BITS>
__global__ void __launch_bounds__(kProcThreads, 5) fused_kernel(const __grid_constant__ ProcArgs a) {
  extern __shared__ uint4 smem[];
  const int64_t row = blockIdx.x;
  const TI* in = (const TI*)a.in + row * a.in_stride;
  TO* out = (TO*)a.out + row * a.out_stride;
  const RowMask mask = row_mask(a.r, row, a.status, threadIdx.x == 0);
  stream_slice<TI, TO>(a, in, out, 0, mask);
  penalise<TI, TO, BITS, false>(a, in, out, row, 0, mask, smem, [] {});  // its barriers order the stores
}

template <typename TI, typename TO, int BITS, bool HASH>
__global__ void __launch_bounds__(kCountThreads, 2) penalise_kernel(const __grid_constant__ ProcArgs a) {
  extern __shared__ uint4 smem[];
  const int64_t row = blockIdx.x >> a.lg;
  const RowMask mask = row_mask(a.r, row, a.status, false);
  // in place, streaming writes -inf to what the mask excludes: those logits are not used here
  penalise<TI, TO, BITS, HASH>(a, (const TI*)a.in + row * a.in_stride, (TO*)a.out + row * a.out_stride, row,
                               (int)(blockIdx.x & ((1u << a.lg) - 1)), mask, smem,
                               [] { asm volatile("griddepcontrol.wait;" ::: "memory"); });
}

// Lets a kernel have more than 48 KB of shared memory: always `most`, so that
// calls of other sizes in other threads never set a lower limit in between.
template <typename F>
int allow_smem(F* kernel, size_t smem, int most) {
  if (smem > (size_t)most) return set_error(CNNUE_ERR_INVALID_ARG, "%zu bytes of shared memory", smem);
  if (smem > 40 * 1024) CNNUE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
  return CNNUE_OK;
}

template <typename F>
int launch_process(F* kernel, const ProcArgs& a, int64_t blocks, int threads, size_t smem, bool dependent, cudaStream_t s,
                   const char* what) {
  if (blocks > 0x7fffffff) return set_error(CNNUE_ERR_INVALID_ARG, "too many rows for one call");
  if (int st = allow_smem(kernel, smem, kCountBytes)) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  CNNUE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return check_launch_error(what);
}

// Vectors that cover a row: one more only where a row may start inside one.
template <typename T>
int64_t row_vectors(const void* p, int64_t stride, int64_t vocab) {
  constexpr int VE = Vec<T>::VE;
  return (uintptr_t)p % 16 == 0 && stride % VE == 0 ? (vocab + VE - 1) / VE : rows::max_vectors<T>(vocab);
}

template <typename TI, typename TO>
int pick_process(ProcArgs& a, int64_t n_rows, cudaStream_t s) {
  const int64_t nv = row_vectors<TI>(a.in, a.in_stride, a.vocab);
  // a history without penalties changes nothing, but its tokens and lengths are checked all the same
  if (!a.r.history || (a.r.history_len == 0 && !a.r.lengths)) {
    a.r.history = nullptr;
    a.r.history_len = 0;
  }
  if (a.r.bias_count == 0) a.r.bias_tokens = nullptr;
  const bool count = a.r.history || a.r.bias_tokens, bias = a.r.bias_tokens != nullptr, wide = a.r.history_len > 32767;
  const int64_t len = a.r.history_len;
  auto per_thread = [](int64_t n, int each, int most) {  // threads for n items
    return (int)std::min<int64_t>(most, std::max<int64_t>(1, n / (each * 32)) * 32);
  };
  if (count && a.vocab <= kFusedTokens) {
    a.split = 1, a.vps = (int)nv, a.slots = a.vocab, a.lg = 0;
    const int threads = per_thread(nv, kProcAhead, kProcThreads);
    return wide ? launch_process(fused_kernel<TI, TO, 32>, a, n_rows, threads,
                                 Table<32, false>::bytes(a.slots, bias, len), false, s, "fused_kernel")
                : launch_process(fused_kernel<TI, TO, 16>, a, n_rows, threads,
                                 Table<16, false>::bytes(a.slots, bias, len), false, s, "fused_kernel");
  }
  const bool stream = !a.in_place || a.r.mask;
  if (stream) {
    a.vps = (int)std::min<int64_t>(nv, 2 * kProcAhead * kProcThreads);
    a.split = (int)((nv + a.vps - 1) / a.vps);
    if (int st = launch_process(stream_kernel<TI, TO>, a, n_rows * a.split, per_thread(a.vps, kProcAhead, kProcThreads), 0,
                                false, s, "stream_kernel"))
      return st;
  }
  if (!count) return CNNUE_OK;
  const int64_t named = len + a.r.bias_count;
  if (len <= kHashTokens && named <= 2 * kHashTokens) {
    a.lg = 0;
    a.slots = 64;
    while (a.slots < 2 * named) a.slots *= 2;
    const int threads = len <= 128 * kTokensAhead ? 128 : len <= 256 * kTokensAhead ? 256 : kCountThreads;
    return launch_process(penalise_kernel<TI, TO, 16, true>, a, n_rows, threads, Table<16, true>::bytes(a.slots, bias, len),
                          stream, s, "penalise_kernel");
  }
  const int64_t most = wide ? 16384 : 32768;  // 64 KB of counters
  a.lg = 0;
  while (((int64_t)a.vocab + (1 << a.lg) - 1) >> a.lg > most) ++a.lg;
  a.slots = (int)(((int64_t)a.vocab + (1 << a.lg) - 1) >> a.lg);
  return wide ? launch_process(penalise_kernel<TI, TO, 32, false>, a, n_rows << a.lg, kCountThreads,
                               Table<32, false>::bytes(a.slots, bias, len), stream, s, "penalise_kernel")
              : launch_process(penalise_kernel<TI, TO, 16, false>, a, n_rows << a.lg, kCountThreads,
                               Table<16, false>::bytes(a.slots, bias, len), stream, s, "penalise_kernel");
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

struct LossArgs {
  const void* z;
  int64_t z_stride;
  int vocab;
  int split, vps;         // slices (CTAs) per row, vectors per slice
  int64_t n_rows;
  cnnue_loss_targets t;
  const float* upstream;  // [rows] or null (backward pass)
  float* loss;            // [rows] or null
  float* stats;           // [rows][3]: M, S, T (written by the forward pass, read by the backward pass)
  void* grad;
  int64_t grad_stride;
  uint32_t* status;
};

// Exponentials are exp2(x c - B) with c = log2(e) in fp32 and B = m c rounded:
// one fused operation per element before the instruction, and because every
// thread and both passes take the same B for the same m, B's rounding r = m c -
// B cancels in exp / sum; the loss takes it out (residual()).  Above |m| = 2^16,
// where r is no longer small (2^-8 there) and m c in the end overflows, they
// are exp2((x - m) c), and r is 0.
struct Sums {
  float m, s, t, d;  // maximum, sum of exp2(z c - B(m)), target mass, sum of t (m - z)
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ bool huge(float m) { return fabsf(m) > 65536.f; }  // infinities too
__device__ __forceinline__ float base(float m) { return __fmul_rn(m, rows::kLog2e); }
__device__ __forceinline__ float rounding(float m) { return huge(m) ? 0.f : fmaf(m, rows::kLog2e, -base(m)); }
// exp2(z c - B(from)) times this is exp2(z c - B(to)); from -inf: 0.
__device__ __forceinline__ float rebase(float from, float to) {
  if (from == kNegInf) return 0.f;
  if (huge(from) || huge(to)) return exp2_fast((from - to) * rows::kLog2e - rounding(from) + rounding(to));
  return exp2_fast(base(from) - base(to));
}
// log of what B's rounding put into the sum.
__device__ __forceinline__ float residual(float m) { return 0.693147180559945309f * rounding(m); }
// exp2(z c - B(m)) of one logit, m not -inf.
__device__ __forceinline__ float exp_of(float z, float m) {
  return exp2_fast(huge(m) ? (z - m) * rows::kLog2e : fmaf(z, rows::kLog2e, -base(m)));
}
// What a move of the maximum to m, not -inf, adds to d.  Masses that cancel (t =
// 0) leave d as it is: a sum of signed terms, not 0.  So do those of a side
// without a logit above -inf: each is t inf there already, as t (m - z) says.
__device__ __forceinline__ float moved(const Sums& v, float m) {
  return v.t != 0.f && v.m != kNegInf ? v.t * (m - v.m) : 0.f;
}
// The sums of the warp's lanes, each relative to its own maximum, as one;
// every lane gets the same bits.  A side without a logit above -inf has s = 0.
// TARGETS: t and d too (otherwise they are 0 in every lane).
__device__ __forceinline__ Sums join_lanes(Sums v, bool targets) {
  float m;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v.m));
  if (m != kNegInf) {
    v.s *= rebase(v.m, m);
    if (targets) v.d += moved(v, m);
  }
  v.m = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) v.s += __shfl_xor_sync(~0u, v.s, o);
  if (targets) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      v.t += __shfl_xor_sync(~0u, v.t, o);
      v.d += __shfl_xor_sync(~0u, v.d, o);
    }
  }
  return v;
}
// a += b, each relative to its own maximum.
__device__ __forceinline__ void join_two(Sums& a, const Sums& b) {
  const float m = rows::max_nan(a.m, b.m);
  if (m != kNegInf) {
    a.s = a.s * rebase(a.m, m) + b.s * rebase(b.m, m);
    a.d += b.d + moved(a, m) + moved(b, m);
  }
  a.t += b.t;
  a.m = m;
}
__device__ __forceinline__ Sums nothing() { return {kNegInf, 0.f, 0.f, 0.f}; }

constexpr int kLossThreads = 256;
constexpr int kLossWarps = kLossThreads / 32;
constexpr int kMaxCluster = 8;  // the portable size
static_assert(kLossWarps * kMaxCluster <= 64, "two warps' sums per lane");

// The sums of a row: every warp's go into its CTA's `shared`, and after one
// barrier (of the cluster, if the row has one) every warp joins those of all
// warps of the row, over distributed shared memory, in the same order.
// `targets`: this warp has target sums.  The caller waits for the cluster
// (cluster_done) before it leaves.
__device__ __forceinline__ Sums join_all(Sums v, bool targets, Sums* shared, int ctas) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v = join_lanes(v, targets);
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  if (ctas > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    // lane l: warp l % 8 of CTAs l / 8 and 4 + l / 8
    v = nothing();
    if ((lane & 7) < warps && lane / 8 < ctas) v = cluster.map_shared_rank(shared, lane / 8)[lane & 7];
    if (ctas > 4 && (lane & 7) < warps) join_two(v, cluster.map_shared_rank(shared, 4 + lane / 8)[lane & 7]);
    v = join_lanes(v, true);
    // nothing is handed over: it only keeps this CTA's shared memory until all have read it
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  } else {
    __syncthreads();
    if (warps > 1) v = join_lanes(lane < warps ? shared[lane] : nothing(), true);
  }
  return v;
}
__device__ __forceinline__ void cluster_done(int ctas) {
  if (ctas > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// One row's tensors as a CTA sees them.
template <typename T>
struct LossRow {
  static constexpr int VE = Vec<T>::VE;
  const LossArgs* args;
  int64_t row;
  const T* z;
  int shift;
  RowMask mask;
  const char* list;
  const float* prob;
  bool wide;

  __device__ __forceinline__ LossRow(const LossArgs& a, int64_t r, bool tell) : args(&a), row(r) {
    z = (const T*)a.z + row * a.z_stride;
    shift = rows::shift_of(z);
    mask = row_mask(a.t, row, a.status, tell);
    wide = a.t.index_bytes == 8;
    list = a.t.index ? (const char*)a.t.index + row * a.t.index_stride * a.t.index_bytes : nullptr;
    prob = a.t.prob ? a.t.prob + row * a.t.prob_stride : nullptr;
  }
  __device__ __forceinline__ uint32_t allowed(int e0, bool whole) const {
    if (whole) return mask.dead ? 0 : mask.words ? rows::allowed_whole<VE>(mask.words, e0) : rows::kFull<VE>;
    return mask.dead ? 0 : mask.words ? rows::allowed<VE>(mask.words, e0, args->vocab) : rows::inside<VE>(e0, args->vocab);
  }
  // The dense targets of vector e0 (whole: it lies inside the row), 0 where
  // `ok` has no bit.
  __device__ __forceinline__ void targets(int e0, uint32_t ok, bool whole, float* t) const {
    const int64_t at = row * args->t.dense_stride + e0;
    if (args->t.dense_type == CNNUE_F32)
      dense_vec<float>(at, ok, whole, t);
    else if (args->t.dense_type == CNNUE_BF16)
      dense_vec<__nv_bfloat16>(at, ok, whole, t);
    else
      dense_vec<__half>(at, ok, whole, t);
  }
  template <typename D>
  __device__ __forceinline__ void dense_vec(int64_t at, uint32_t ok, bool whole, float* t) const {
    constexpr int DE = Vec<D>::VE;
    const D* p = (const D*)args->t.dense + at;
    if (whole && VE % DE == 0 && ((uintptr_t)p & 15) == 0) {  // the targets' vectors line up with the logits'
#pragma unroll
      for (int j = 0; j < VE / DE; ++j) Vec<D>::unpack(__ldg(reinterpret_cast<const uint4*>(p) + j), t + j * DE);
      if (ok != rows::kFull<VE>) {
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (!(ok >> i & 1)) t[i] = 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) t[i] = ok >> i & 1 ? Vec<D>::up(p[i]) : 0.f;
    }
  }
  // Entry k of the list: its token, or -1 when it does not count.
  __device__ __forceinline__ int entry(int64_t k) const {
    const int tok = rows::token_at(list, k, wide);
    return tok >= 0 && tok < args->vocab && token_ok(mask, tok) ? tok : -1;
  }
  __device__ __forceinline__ float mass(int64_t k) const { return prob ? __ldg(prob + k) : 1.f; }

  template <bool DENSE>
  __device__ void edge_grad(int e0, bool none, T* g, float m, float c, float w) const;

  // Mass and d of the list's entries on tokens [lo, hi), relative to v.m;
  // repeated tokens are marked.
  __device__ __forceinline__ void list_sums(int lo, int hi, bool tell, Sums& v, Repeats& repeats) const {
    for (int64_t k = threadIdx.x; k < args->t.count; k += blockDim.x) {
      if (tell && rows::token_at(list, k, wide) >= args->vocab) atomicOr(args->status, CNNUE_STATUS_BAD_INDEX);
      const int tok = entry(k);
      if (tok < lo || tok >= hi) continue;
      if (args->t.count > 1) repeats.mark(tok);
      const float t = mass(k);
      if (t == 0.f) continue;
      const float x = Vec<T>::up(z[tok]);
      // relative to this thread's own maximum, which need not be above x
      if (v.m == kNegInf) v.m = x;  // s = 0
      v.t += t;
      v.d += t * ((v.m == kNegInf ? 0.f : v.m) - x);  // t inf on a logit of -inf
    }
  }

  // The gradient at the listed tokens [lo, hi): c exp(z - m) - w t.  A token
  // that may be listed more than once is summed in list order by the thread of
  // its first entry (every thread walks the whole list, so that a warp's lanes
  // stay together).
  __device__ __forceinline__ void list_grads(int lo, int hi, T* g, float m, float c, float w, const Repeats& repeats) const {
    for (int64_t k = threadIdx.x; k < args->t.count; k += blockDim.x) {
      const int tok = entry(k);
      if (tok < lo || tok >= hi) continue;
      float t;
      if (args->t.count == 1 || !repeats.marked(tok)) {
        t = mass(k);
      } else {
        t = 0.f;
        bool earlier = false;
        for (int64_t j = 0; j < args->t.count; ++j) {
          if (rows::token_at(list, j, wide) != tok) continue;
          earlier |= j < k;
          t += mass(j);
        }
        if (earlier) continue;
      }
      g[tok] = Vec<T>::down((c == 0.f ? 0.f : c * exp_of(Vec<T>::up(z[tok]), m)) - w * t);
    }
  }
};

// exp2(x c - B(m)) of a vector, m not -inf; *sum gets their sum.
template <int VE>
__device__ __forceinline__ void exps(float* x, float m, float2* sum) {
  if (!huge(m)) {
    const float2 c = make_float2(rows::kLog2e, rows::kLog2e), minus = make_float2(-base(m), -base(m));
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
      const float2 d = rows::fma2(make_float2(x[j], x[j + 1]), c, minus);
      x[j] = exp2_fast(d.x);
      x[j + 1] = exp2_fast(d.y);
    }
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) x[j] = exp2_fast((x[j] - m) * rows::kLog2e);
  }
  if (sum) {
#pragma unroll
    for (int j = 0; j < VE; j += 2) *sum = rows::add2(*sum, make_float2(x[j], x[j + 1]));
  }
}
// The gradient's vector e0 from the raw logits: c exp2(z c' - B(m)) - w t on
// `ok`, 0 elsewhere.  c = 0: nothing but the targets (and the logits are not
// looked at, so no NaN comes from them).
template <typename T, bool DENSE>
__device__ __forceinline__ void grad_vector(const LossRow<T>& r, const uint4& raw, int e0, uint32_t ok, bool whole, float m,
                                            float c, float w, float* x) {
  constexpr int VE = Vec<T>::VE;
  if (c != 0.f && ok) {
    Vec<T>::unpack(raw, x);
    exps<VE>(x, m, nullptr);
#pragma unroll
    for (int j = 0; j < VE; j += 2) {
      const float2 e = rows::mul2(make_float2(x[j], x[j + 1]), make_float2(c, c));
      x[j] = e.x;
      x[j + 1] = e.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j) x[j] = 0.f;
  }
  if (DENSE && ok) {
    float t[VE];
    r.targets(e0, ok, whole, t);
#pragma unroll
    for (int j = 0; j < VE; ++j) x[j] -= w * t[j];
  }
  if (ok != rows::kFull<VE>) {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (!(ok >> j & 1)) x[j] = 0.f;
  }
}

// The gradient of a row's partial vector.
template <typename T>
template <bool DENSE>
__device__ __forceinline__ void LossRow<T>::edge_grad(int e0, bool none, T* g, float m, float c, float w) const {
  const uint32_t in = rows::inside<VE>(e0, args->vocab), ok = none ? 0 : allowed(e0, false);
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (c != 0.f && ok) raw = rows::load_raw(z, e0, in, ok);
  float x[VE];
  grad_vector<T, DENSE>(*this, raw, e0, ok, false, m, c, w, x);
  rows::store<T, VE>(g, e0, in, false, x);
}

constexpr int kTogether = 4;  // vectors per thread in the gradient loop
constexpr int kAhead = 4;     // vectors per thread between two looks at the running maximum

// The sums of one slice, relative to each thread's running maximum.  KEEP: the
// whole vectors lie in `kept`.
template <typename T, bool KEEP, bool DENSE>
__device__ __forceinline__ Sums slice_sums(const LossRow<T>& r, const Slice<Vec<T>::VE>& slice, const uint4* kept) {
  constexpr int VE = Vec<T>::VE;
  const int stride = blockDim.x;
  Sums v = nothing();
  float2 sum = make_float2(0.f, 0.f);
  // raw[N] with -inf where nothing is allowed, ok[N]: the vectors at e0 + j stride VE
  auto add = [&](const uint4* raw, const uint32_t* ok, int e0, bool whole, auto n) {
    constexpr int N = decltype(n)::value;
    float m = Vec<T>::top(raw[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) m = rows::max_nan(m, Vec<T>::top(raw[j]));
    if (!(m <= v.m)) {  // a new maximum, or a NaN: what is summed so far relative to it
      m = rows::max_nan(m, v.m);  // a NaN stays one, whatever follows it
      const float f = rebase(v.m, m);
      sum.x *= f;
      sum.y *= f;
      v.d += moved(v, m);
      v.m = m;
    }
    const float from = v.m == kNegInf ? 0.f : v.m;  // -inf - -inf would be a NaN
#pragma unroll
    for (int j = 0; j < N; ++j) {
      float x[VE];
      Vec<T>::unpack(raw[j], x);
      if (DENSE && ok[j]) {
        float t[VE];
        r.targets(e0 + j * stride * VE, ok[j], whole, t);
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          v.t += t[k];
          if (t[k] != 0.f) v.d += t[k] * (from - x[k]);
        }
      }
      exps<VE>(x, from, &sum);
    }
  };
  slice.template each<kAhead>([&](int i, int e0, auto n) {
    constexpr int N = decltype(n)::value;
    uint4 raw[N];
    uint32_t ok[N];
    if (!r.args->t.mask) {  // nothing to look out for
#pragma unroll
      for (int j = 0; j < N; ++j) {
        ok[j] = rows::kFull<VE>;
        raw[j] = KEEP ? kept[i + j * stride] : rows::load16(r.z + e0 + j * stride * VE);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        ok[j] = r.allowed(e0 + j * stride * VE, true);
        raw[j] = make_uint4(0, 0, 0, 0);
        if (ok[j]) raw[j] = KEEP ? kept[i + j * stride] : rows::load16(r.z + e0 + j * stride * VE);
      }
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (ok[j] != rows::kFull<VE>) raw[j] = Vec<T>::only(raw[j], ok[j]);
    }
    add(raw, ok, e0, true, n);
  });
  slice.edges([&](int e0) {
    const uint32_t in = rows::inside<VE>(e0, r.args->vocab), ok = r.allowed(e0, false);
    const uint4 raw = Vec<T>::only(rows::load_raw(r.z, e0, in, ok), ok);
    add(&raw, &ok, e0, false, std::integral_constant<int, 1>{});
  });
  v.s = sum.x + sum.y;
  return v;
}

// The gradient of one slice from the row's sums, without the lists' targets.
template <typename T, bool KEEP, bool DENSE>
__device__ __forceinline__ void slice_grads(const LossRow<T>& r, const Slice<Vec<T>::VE>& slice, const uint4* kept, T* g,
                                            const Sums& v, bool none, float c, float w) {
  constexpr int VE = Vec<T>::VE;
  const bool lines_up = rows::lines_up(g, r.shift);
  if (!DENSE && KEEP && c != 0.f && !r.args->t.mask && !huge(v.m) && lines_up) {  // nothing to look out for
    const float2 scale = make_float2(rows::kLog2e, rows::kLog2e), minus = make_float2(-base(v.m), -base(v.m));
    const float2 cc = make_float2(c, c);
    const int stride = blockDim.x;
    slice.template each<kTogether>([&](int i, int e0, auto n) {
      constexpr int N = decltype(n)::value;
      uint4 raw[N];
#pragma unroll
      for (int k = 0; k < N; ++k) raw[k] = kept[i + k * stride];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float x[VE];
        Vec<T>::unpack(raw[k], x);
#pragma unroll
        for (int j = 0; j < VE; j += 2) {
          float2 d = rows::fma2(make_float2(x[j], x[j + 1]), scale, minus);
          d = rows::mul2(make_float2(exp2_fast(d.x), exp2_fast(d.y)), cc);
          x[j] = d.x, x[j + 1] = d.y;
        }
        *reinterpret_cast<uint4*>(g + e0 + k * stride * VE) = Vec<T>::pack(x);
      }
    });
  } else {
    slice.template each<1>([&](int i, int e0, auto) {
      const uint32_t ok = none ? 0 : r.allowed(e0, true);
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (c != 0.f && ok) raw = KEEP ? kept[i] : rows::load16(r.z + e0);
      float x[VE];
      grad_vector<T, DENSE>(r, raw, e0, ok, true, v.m, c, w, x);
      rows::store<T, VE>(g, e0, rows::kFull<VE>, lines_up, x);
    });
  }
  slice.edges([&](int e0) { r.template edge_grad<DENSE>(e0, none, g, v.m, c, w); });
}

// Loss, and with GRAD the gradient, of one slice of a row; the slices of a row
// are the CTAs of a cluster.  A thread takes every blockDim-th vector of the
// slice.  KEEP: it copies them into shared memory, all in flight at once, and
// reads them there twice, for the row's sums and, once the cluster has joined
// those, for the gradient: the row is read from memory once, and some 200 KB
// per SM are in flight.  A slot is written and read by one thread: no barrier.
// Otherwise (rows that do not fit, or no gradient) the vectors come from
// memory, or L2, each time.  4096 x 131072 bf16 with labels: 435 us, 72 - 75 %
// of the copy rate; without the barrier and the joins 1024 rows took 101 us of
// 135, so it is the wait between the two readings that bounds it, with 24
// warps per SM around it.
template <typename T, bool KEEP, bool GRAD, bool DENSE>
__global__ void __launch_bounds__(kLossThreads, 4) loss_kernel(const __grid_constant__ LossArgs a) {
  __shared__ Sums shared[kLossWarps];
  __shared__ Repeats repeats;
  extern __shared__ uint4 kept[];
  const int rank = (int)(blockIdx.x & (a.split - 1));  // split: a power of two
  const int64_t row = blockIdx.x >> (31 - __clz(a.split));
  const LossRow<T> r(a, row, threadIdx.x == 0 && rank == 0);
  const Slice<Vec<T>::VE> slice(rank, a.vps, r.shift, a.vocab);
  const float w = a.t.weights ? a.t.weights[row] : 1.f;
  const bool idle = w == 0.f;  // a padded row: not read, loss and gradient 0
  const bool lists = !DENSE && a.t.count > 1;

  Sums v = nothing();
  if (!idle) {
    if (KEEP) {
      slice.template each<1>([&](int i, int e0, auto) {
        if (r.allowed(e0, true))
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(kept + i)),
                       "l"(r.z + e0)
                       : "memory");
      });
      if (lists) repeats.clear();
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (lists) {
      repeats.clear();
    }
    v = slice_sums<T, KEEP, DENSE>(r, slice, kept);
    if (lists) __syncthreads();  // cleared
    bool targets = DENSE;
    if (!DENSE) {  // the list's sums: by as few warps as its length needs
      const bool mine = (threadIdx.x & ~31) < a.t.count;
      if (mine) r.list_sums(slice.lo, slice.hi, rank == 0, v, repeats);
      targets = mine;
    }
    v = join_all(v, targets, shared, a.split);
  }
  const bool none = v.m == kNegInf;  // nothing is left of the row
  if (rank == 0 && threadIdx.x == 0) {
    if (a.loss) a.loss[row] = none ? 0.f : w * (v.t * (logf(v.s) - residual(v.m)) + v.d);
    if (a.stats) {
      a.stats[3 * row] = v.m;
      a.stats[3 * row + 1] = v.s;
      a.stats[3 * row + 2] = v.t;
    }
  }
  if (GRAD) {
    T* g = (T*)a.grad + row * a.grad_stride;
    const float c = none ? 0.f : w * v.t / v.s;  // without target mass 0, or a NaN that s holds
    slice_grads<T, KEEP, DENSE>(r, slice, kept, g, v, none, c, w);
    if (!DENSE && !none) {
      __syncthreads();  // the listed tokens' elements again, now with their targets
      r.list_grads(slice.lo, slice.hi, g, v.m, c, w, repeats);
    }
  }
  if (!idle) cluster_done(a.split);
}

// The gradient from the sums of an earlier forward pass; the slices of a row
// are independent CTAs.
template <typename T, bool DENSE>
__global__ void __launch_bounds__(kLossThreads) loss_bwd_kernel(const LossArgs a) {
  constexpr int VE = Vec<T>::VE;
  const int rank = (int)(blockIdx.x % a.split);
  const LossRow<T> r(a, blockIdx.x / a.split, threadIdx.x == 0 && rank == 0);
  float w = a.t.weights ? a.t.weights[r.row] : 1.f;
  const float m = a.stats[3 * r.row], s = a.stats[3 * r.row + 1], mass = a.stats[3 * r.row + 2];
  const bool none = w == 0.f || m == kNegInf;
  if (a.upstream) w *= a.upstream[r.row];
  const float c = none ? 0.f : w * mass / s;
  const Slice<VE> slice(rank, a.vps, r.shift, a.vocab);
  __shared__ Repeats repeats;
  if (!DENSE && !none && a.t.count > 1) {
    repeats.clear();
    __syncthreads();
    for (int64_t k = threadIdx.x; k < a.t.count; k += blockDim.x) {
      const int tok = r.entry(k);
      if (tok >= slice.lo && tok < slice.hi) repeats.mark(tok);
    }
  }
  T* g = (T*)a.grad + r.row * a.grad_stride;
  const bool lines_up = rows::lines_up(g, r.shift);
  slice.template each<kAhead>([&](int, int e0, auto n) {
    constexpr int N = decltype(n)::value;
    uint4 raw[N];
    uint32_t ok[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = e0 + j * (int)blockDim.x * VE;
      ok[j] = none ? 0 : r.allowed(e, true);
      raw[j] = make_uint4(0, 0, 0, 0);
      if (c != 0.f && ok[j]) raw[j] = rows::load16(r.z + e);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = e0 + j * (int)blockDim.x * VE;
      float x[VE];
      grad_vector<T, DENSE>(r, raw[j], e, ok[j], true, m, c, w, x);
      rows::store<T, VE>(g, e, rows::kFull<VE>, lines_up, x);
    }
  });
  slice.edges([&](int e0) { r.template edge_grad<DENSE>(e0, none, g, m, c, w); });
  if (!DENSE && !none) {
    __syncthreads();
    r.list_grads(slice.lo, slice.hi, g, m, c, w, repeats);
  }
}

// A slice is at most 64 KB of shared memory, 3 CTAs per SM.  Measured at 1024 x
// 131072 bf16: 117 us with 4 CTAs of 64 KB per row, 139 with 8 of 32 KB (twice
// the threads' fixed work, and more to wait for in each cluster).
constexpr int kSliceVectors = 4096;
// Longer rows keep slices of up to 100 KB, 2 CTAs per SM (400 x 200000 fp32:
// 152 us, 196 read twice).  Above that one CTA fills an SM: slower than reading
// twice when the clusters take turns (dense 16 x 262144 fp32: 107 us, 87; 600
// rows: 428, 338), faster while all run at once (14 rows: 66 us, 87), which 14
// clusters of 8 do; up to 192 KB.
constexpr int kKeepVectors = 6400, kKeepAlone = 12288, kAloneCtas = 112;

template <typename T, bool KEEP, bool GRAD, bool DENSE>
int launch_loss(const LossArgs& a, int threads, cudaStream_t s) {
  if (a.n_rows * a.split > 0x7fffffff) return set_error(CNNUE_ERR_INVALID_ARG, "too many rows for one call");
  auto* kernel = loss_kernel<T, KEEP, GRAD, DENSE>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_rows * a.split));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = KEEP ? (size_t)a.vps * 16 : 0;
  cfg.stream = s;
  if (int st = allow_smem(kernel, cfg.dynamicSmemBytes, kKeepAlone * 16)) return st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)a.split, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = a.split > 1 ? 1 : 0;
  CNNUE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  return check_launch_error("loss_kernel");
}

template <typename T, bool GRAD>
int run_loss(LossArgs a, cudaStream_t s) {
  const int64_t nv = row_vectors<T>(a.z, a.z_stride, a.vocab);
  int64_t ctas = 1;
  while (ctas < kMaxCluster && nv > kSliceVectors * ctas) ctas *= 2;
  a.split = (int)ctas;
  a.vps = (int)((nv + ctas - 1) / ctas);
  // Vectors per thread: 4 while all CTAs run at once anyway and latency counts (1024 x 2086 fp32 dense: 13.4 us, 17.1
  // with 8), 8 for more rows, where the threads' fixed work counts (16384 x 2086 fp32: 66 us, 82 with 4).
  const int per = a.n_rows * ctas > 148 * 8 ? 8 : 4;
  const int threads = (int)std::min<int64_t>(kLossThreads, std::max<int64_t>(1, a.vps / (per * 32)) * 32);
  if (GRAD && a.vps <= (a.n_rows * ctas <= kAloneCtas ? kKeepAlone : kKeepVectors))
    return a.t.dense ? launch_loss<T, GRAD, GRAD, true>(a, threads, s) : launch_loss<T, GRAD, GRAD, false>(a, threads, s);
  return a.t.dense ? launch_loss<T, false, GRAD, true>(a, threads, s) : launch_loss<T, false, GRAD, false>(a, threads, s);
}

template <typename T>
int run_loss_bwd(LossArgs a, int64_t n_rows, cudaStream_t s) {
  constexpr int NV = 4;
  const int64_t nv = row_vectors<T>(a.z, a.z_stride, a.vocab);
  a.vps = (int)std::min<int64_t>(nv, NV * kLossThreads);
  a.split = (int)((nv + a.vps - 1) / a.vps);
  const int threads = (int)std::min<int64_t>(kLossThreads, (a.vps + NV * 32 - 1) / (NV * 32) * 32);
  if (n_rows * a.split > 0x7fffffff) return set_error(CNNUE_ERR_INVALID_ARG, "too many rows for one call");
  if (a.t.dense)
    loss_bwd_kernel<T, true><<<(unsigned)(n_rows * a.split), threads, 0, s>>>(a);
  else
    loss_bwd_kernel<T, false><<<(unsigned)(n_rows * a.split), threads, 0, s>>>(a);
  return check_launch_error("loss_bwd_kernel");
}

template <bool FWD, bool GRAD>
int pick_loss(const LossArgs& a, int type, int64_t n_rows, cudaStream_t s) {
  if (!FWD)
    return type == CNNUE_F32    ? run_loss_bwd<float>(a, n_rows, s)
           : type == CNNUE_BF16 ? run_loss_bwd<__nv_bfloat16>(a, n_rows, s)
                                : run_loss_bwd<__half>(a, n_rows, s);
  return type == CNNUE_F32    ? run_loss<float, GRAD>(a, s)
         : type == CNNUE_BF16 ? run_loss<__nv_bfloat16, GRAD>(a, s)
                              : run_loss<__half, GRAD>(a, s);
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

int check_mask(const uint32_t* mask, int64_t stride, int64_t mask_rows, const int32_t* index, int64_t n_rows) {
  if (!mask) return index ? set_error(CNNUE_ERR_INVALID_ARG, "mask_index without a mask") : CNNUE_OK;
  if (mask_rows < 0 || stride < 0) return set_error(CNNUE_ERR_INVALID_ARG, "mask: rows or stride");
  if (!index && mask_rows != 1 && mask_rows != n_rows)
    return set_error(CNNUE_ERR_INVALID_ARG, "mask: %lld rows for %lld rows of logits", (long long)mask_rows,
                     (long long)n_rows);
  return CNNUE_OK;
}

// Whether the two row sets share a byte.  Rows at the same distance may lie
// between each other's, as two column ranges of one matrix do.
bool overlap(const void* p, int64_t p_stride, int pb, const void* q, int64_t q_stride, int qb, int64_t n_rows,
             int64_t vocab) {
  const uintptr_t p0 = (uintptr_t)p, p1 = p0 + ((n_rows - 1) * p_stride + vocab) * pb;
  const uintptr_t q0 = (uintptr_t)q, q1 = q0 + ((n_rows - 1) * q_stride + vocab) * qb;
  if (p1 <= q0 || q1 <= p0) return false;
  const int64_t step = p_stride * pb;
  if (n_rows == 1 || step == 0 || step != q_stride * qb || vocab * pb > step) return true;
  const int64_t apart = ((int64_t)(q0 - p0) % step + step) % step;  // from a row of p to the next row of q
  return apart < vocab * pb || apart + vocab * qb > step;
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
  return check_mask(t->mask, t->mask_stride, t->mask_rows, t->mask_index, n_rows);
}

// The gradient may share memory with neither the logits nor dense targets:
// both are read again after parts of it are written.
int check_grad(const void* grad, int64_t grad_stride, const void* z, int64_t z_stride, int type, const cnnue_loss_targets* t,
               int64_t n_rows, int64_t vocab) {
  if (int st = check_rows(grad, grad_stride, type, n_rows, vocab, true, "grad")) return st;
  const int b = element_bytes(type);
  if (overlap(z, z_stride, b, grad, grad_stride, b, n_rows, vocab))
    return set_error(CNNUE_ERR_INVALID_ARG, "grad overlaps the logits");
  if (t->dense && overlap(t->dense, t->dense_stride, element_bytes(t->dense_type), grad, grad_stride, b, n_rows, vocab))
    return set_error(CNNUE_ERR_INVALID_ARG, "grad overlaps the targets");
  return CNNUE_OK;
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
    if (r.history_len < 0 || r.history_len > kMostTokens || r.history_stride < 0)
      return set_error(CNNUE_ERR_INVALID_ARG, "history: length or stride");
  } else if (r.repetition || r.frequency || r.presence || r.lengths || r.prompt_lengths) {
    return set_error(CNNUE_ERR_INVALID_ARG, "penalties without a history");
  }
  if ((r.bias_tokens != nullptr) != (r.bias_values != nullptr))
    return set_error(CNNUE_ERR_INVALID_ARG, "bias tokens and values come together");
  if (r.bias_count < 0 || r.bias_count > 0x7fffffff || r.bias_tokens_stride < 0 || r.bias_values_stride < 0)
    return set_error(CNNUE_ERR_INVALID_ARG, "bias: count or stride");
  if (int st = check_mask(r.mask, r.mask_stride, r.mask_rows, r.mask_index, n_rows)) return st;
  ProcArgs a{d_logits, d_out, logits_stride, out_stride, (int)vocab, 0, 0, 0, 0, in_place, r, d_status};
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
  const LossArgs a{d_logits, logits_stride, (int)vocab, 0, 0, n_rows, *targets, nullptr, d_loss, d_stats, nullptr, 0, d_status};
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
  if (int st = check_grad(d_grad, grad_stride, d_logits, logits_stride, logits_type, targets, n_rows, vocab)) return st;
  if (!d_stats) return set_error(CNNUE_ERR_INVALID_ARG, "null stats");
  const LossArgs a{d_logits,   logits_stride, (int)vocab, 0, 0, n_rows, *targets, d_upstream, nullptr, const_cast<float*>(d_stats),
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
  if (int st = check_grad(d_grad, grad_stride, d_logits, logits_stride, logits_type, targets, n_rows, vocab)) return st;
  if (!d_loss) return set_error(CNNUE_ERR_INVALID_ARG, "null loss");
  const LossArgs a{d_logits, logits_stride, (int)vocab, 0, 0, n_rows, *targets, nullptr, d_loss, nullptr, d_grad, grad_stride, d_status};
  return pick_loss<true, true>(a, logits_type, n_rows, (cudaStream_t)stream);
}

}  // extern "C"
