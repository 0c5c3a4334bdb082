// C ABI: log probabilities over a vocabulary that is split over the members of a team, and their
// gradient (rsm_logprob_to_all, rsm_logprob_to_all_grad; no counterpart in the reference).
//
// With x a row's logits over all members, y = c x and m = max y:
//   l = sum exp(y - m)          lse = m + ln l
//   logprob = y[token] - lse    entropy = ln l - sum exp(y - m) (y - m) / l
//   top: the k largest x, equal ones by ascending id, with their log probabilities
// and backwards, with p = exp(y - lse):
//   dx = c (g_logprob (1[token] - p) + g_lse p - g_entropy p (y - lse + entropy))
//
// The forward pass reads every logit once.  A lane keeps a running maximum m of its own x, and
// l = sum 2^((x - m) c2) and w = sum 2^((x - m) c2) (x - m) c2, c2 = c log2(e), against it; when m
// grows by d both shrink by 2^(-d c2).  Differences are taken before they are scaled, so rows whose
// logits are all at the type's lowest value come out as any other row of equal logits.  A logit at
// minus infinity has probability 0 and adds nothing to the entropy; m starts at the lowest finite
// value, not at minus infinity, so that such logits never meet an infinite m.
#include <cmath>

#include "roc_shmem.hpp"
#include "rocshmem_device/rows.hpp"
#include "rows_common.hpp"

using namespace rocshmem;
using namespace rocshmem::detail;

namespace {

constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kFarBelow = -200.f;        // 2^-200 is 0 as a float: stands for minus infinity in products
constexpr int kNoId = 0x7fffffff;

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }

struct LogprobForward {
  int rows, vocab, shard, members, top_k;
  int64_t step, ld;
  float scale;
  const char *logits;
  const int64_t *tokens;
  char *logprob, *entropy, *lse, *top_ids, *top_logprobs;
  // A row is cut into batches (kBatch elements, never across members); workgroup
  // q of `parts` takes its share of them in order.
  int batches_per_member, parts;
  float4 *part_sums;     // [rows][parts]: m, l, w
  float *part_values;    // [rows][parts][top_k]
  int *part_ids;
  unsigned *arrived;     // [rows], a 64-bit word apart, 0 on entry and on return
};

constexpr int kDeep = 4;   // 16-byte vectors of a lane in one batch
template <typename T>
constexpr int kBatch = 64 * kRowVec<T> * kDeep;

// (m, l, w) of a set of logits, as above.
struct Softmax {
  float m, l, w;
};

__device__ __forceinline__ void lift(Softmax &a, float m, float c2) {
  const float d = fmaxf((a.m - m) * c2, kFarBelow), f = exp2_of(d);
  a.w = fmaf(a.l, d, a.w) * f;
  a.l *= f;
  a.m = m;
}

__device__ __forceinline__ Softmax join(Softmax a, Softmax b, float c2) {
  const float m = fmaxf(a.m, b.m);
  lift(a, m, c2);
  lift(b, m, c2);
  return {m, a.l + b.l, a.w + b.w};
}

__device__ __forceinline__ Softmax join_lanes(Softmax a, float c2) {
  lift(a, wave_max(a.m), c2);
  return {a.m, wave_sum(a.l), wave_sum(a.w)};
}

// The best elements seen so far by a wave: lane r holds the one of rank r.
struct TopList {
  float value;
  int id;
  float last_value;   // the element of rank top_k - 1, the same in every lane: what another must beat
  int last_id;
};

__device__ __forceinline__ float lane_value(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

__device__ __forceinline__ bool beats(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }

__device__ __forceinline__ void top_clear(TopList &t) {
  t.value = t.last_value = -INFINITY;
  t.id = t.last_id = kNoId;
}

// One more element, the same in every lane.
__device__ __forceinline__ void top_insert(TopList &t, float value, int id, int top_k) {
  if (!beats(value, id, t.last_value, t.last_id)) return;
  const int rank = __popcll(__ballot(beats(t.value, t.id, value, id)));
  const float up_value = __uint_as_float(from_lower_lane(__float_as_uint(t.value)));
  const int up_id = static_cast<int>(from_lower_lane(static_cast<uint32_t>(t.id)));
  const int lane = lane_id();
  t.value = lane > rank ? up_value : lane == rank ? value : t.value;
  t.id = lane > rank ? up_id : lane == rank ? id : t.id;
  t.last_value = lane_value(t.value, top_k - 1);
  t.last_id = static_cast<int>(__builtin_amdgcn_readlane(t.id, top_k - 1));
}

// Every lane offers one element (`offered` false: none).
__device__ __forceinline__ void top_offer(TopList &t, bool offered, float value, int id, int top_k) {
  uint64_t mask = __ballot(offered && beats(value, id, t.last_value, t.last_id));
  while (mask) {
    const int lane = __builtin_ctzll(mask);
    mask &= mask - 1;
    top_insert(t, lane_value(value, lane), static_cast<int>(__builtin_amdgcn_readlane(id, lane)), top_k);
  }
}

// One batch of a wave: `left` elements of the member's part from `p` on.  Returns the largest of this
// lane's elements.
template <typename T, bool kNt>
__device__ __forceinline__ float take_batch(const T *p, int left, float c2, Softmax &a) {
  constexpr int V = kRowVec<T>;
  constexpr uint32_t kMinusInf = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;
  const int lane = lane_id();
  u32x4 raw[kDeep];
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    const int c = (k * 64 + lane) * V;
    raw[k] = row_load<T, true, kNt>(p + c, left - c, kMinusInf);
  }
  float best = -INFINITY;
#pragma unroll
  for (int k = 0; k < kDeep; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) best = fmaxf(best, row_get<T>(raw[k], e));
  lift(a, fmaxf(a.m, best), c2);
#pragma unroll
  for (int k = 0; k < kDeep; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = (row_get<T>(raw[k], e) - a.m) * c2, f = exp2_of(d);
      a.l += f;
      a.w = fmaf(f, fmaxf(d, kFarBelow), a.w);
    }
  return best;
}

// ---- the likeliest alternatives -----------------------------------------------------------------
//
// While it streams, a lane notes the largest element of every batch.  The k-th largest of 64 disjoint
// groups' maxima is a bound that at least k elements of the row reach, and few more: with 64 groups
// and k = 20 some 24.  Only batches whose noted maximum reaches the bound are read again (from the
// caches), their elements above it are gathered in LDS, and one wave ranks them by (value, id).  The
// price per logit is nothing but the maximum that the softmax needs anyway.  Rows in which more than
// kMaxFound elements reach the bound (equal values, or fewer numbers than k) are gone through once
// more in ascending order of ids, batch by batch, into a sorted list.

constexpr int kMaxFound = 256, kNotes = 16;

// Orders floats as unsigned numbers.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A value, in 16 bits' precision and not above it, that the k largest of the lanes' values reach; minus
// infinity where fewer than k do.
__device__ __forceinline__ float bound_of_lanes(float v, int k) {
  const uint32_t key = order_of(v);
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t with = bound | 1u << bit;
    if (__popcll(__ballot(key >= with)) >= k) bound = with;
  }
  const uint32_t u = bound & 0x80000000u ? bound & 0x7fffffffu : ~bound;
  return bound <= 0x007fffffu ? -INFINITY : __uint_as_float(u);   // below: minus infinity and NaN
}

struct Found {
  int count;
  float value[kMaxFound];
  int id[kMaxFound];
};

__device__ __forceinline__ void found_add(Found &f, float value, int id) {
  const int at = atomicAdd(&f.count, 1);
  if (at < kMaxFound) {
    f.value[at] = value;
    f.id[at] = id;
  }
}

// The best of what was found, sorted, by one wave.
__device__ __forceinline__ TopList found_best(const Found &f, int n, int top_k) {
  TopList t;
  top_clear(t);
  const int lane = lane_id();
  if (n > 64) {
    for (int i = 0; i < n; i += 64)
      top_offer(t, i + lane < n, i + lane < n ? f.value[i + lane] : 0.f, i + lane < n ? f.id[i + lane] : 0, top_k);
    return t;
  }
  const float v = lane < n ? f.value[lane] : -INFINITY;
  const int id = lane < n ? f.id[lane] : kNoId;
  int rank = 0;
  for (int i = 0; i < n; ++i) rank += beats(lane_value(v, i), static_cast<int>(__builtin_amdgcn_readlane(id, i)), v, id);
  if (lane >= n) rank = lane;
  // every lane sends its element to the lane of its rank
  t.value = __uint_as_float(__builtin_amdgcn_ds_permute(rank * 4, __float_as_uint(v)));
  t.id = __builtin_amdgcn_ds_permute(rank * 4, id);
  return t;
}

template <typename T>
__device__ __forceinline__ float logit_of(const LogprobForward &p, int row, int64_t id) {
  const int64_t member = id / p.shard;
  const T *x = reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + (id - member * p.shard);
  if constexpr (sizeof(T) == 4) return *x;
  else return bf16_bits_to_float(*reinterpret_cast<const uint16_t *>(x));
}

// Writes a row's results to every member; called by one whole wave.
template <bool kTop>
__device__ __forceinline__ void finish_row(const LogprobForward &p, int row, Softmax a, TopList t, int64_t token, float of_token) {
  const int lane = lane_id();
  const float log_l = log2f(a.l) * kLn2;
  const bool empty = a.l == 0.f;   // no logit above minus infinity
  const float lse = empty ? -INFINITY : fmaf(p.scale, a.m, log_l);
  const float entropy = empty ? 0.f : fmaf(-kLn2, a.w / a.l, log_l);
  float logprob = 0.f;
  if (token >= p.vocab) {
    if (lane == 0) status_raise(kStatusBadArgument);
    logprob = NAN;
  } else if (token >= 0) {
    logprob = empty ? -INFINITY : fmaf(p.scale, of_token - a.m, -log_l);
  }
  for (int m = lane; m < p.members; m += 64) {
    if (p.logprob) reinterpret_cast<float *>(p.logprob + m * p.step)[row] = logprob;
    if (p.entropy) reinterpret_cast<float *>(p.entropy + m * p.step)[row] = entropy;
    if (p.lse) reinterpret_cast<float *>(p.lse + m * p.step)[row] = lse;
  }
  if constexpr (kTop) {
    if (lane < p.top_k) {
      const int64_t at = static_cast<int64_t>(row) * p.top_k + lane;
      // a row of fewer than k numbers (the others NaN) has no more to name
      const bool none = t.id == kNoId;
      const float lp = none ? NAN : empty ? -INFINITY : fmaf(p.scale, t.value - a.m, -log_l);
      for (int m = 0; m < p.members; ++m) {
        if (p.top_ids) reinterpret_cast<int *>(p.top_ids + m * p.step)[at] = none ? -1 : t.id;
        if (p.top_logprobs) reinterpret_cast<float *>(p.top_logprobs + m * p.step)[at] = lp;
      }
    }
  }
}

constexpr int kMaxWaves = 8, kMaxParts = 16;

// Where a batch of a row lies: its first element, how many there are, and the first one's id.
template <typename T>
struct Batch {
  const T *p;
  int left, id;
};
template <typename T>
__device__ __forceinline__ Batch<T> batch_at(const LogprobForward &p, int row, int b) {
  const int member = uniform(b / p.batches_per_member);
  const int at = (b - member * p.batches_per_member) * kBatch<T>;
  const int64_t id = static_cast<int64_t>(member) * p.shard + at;
  int left = p.shard - at;
  if (id + left > p.vocab) left = id < p.vocab ? static_cast<int>(p.vocab - id) : 0;
  return {reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + at, left, static_cast<int>(id)};
}

template <typename T>
__device__ __forceinline__ float element_at(const Batch<T> &b, int c) {
  if constexpr (sizeof(T) == 4) return c < b.left ? b.p[c] : -INFINITY;
  else return c < b.left ? bf16_bits_to_float(reinterpret_cast<const uint16_t *>(b.p)[c]) : -INFINITY;
}

// 64 vector registers at most, so that a compute unit holds four workgroups: while some rank their
// row's alternatives the others stream.
template <typename T, bool kTop, bool kNt>
__global__ void __launch_bounds__(kMaxWaves * 64, 8) logprob_kernel(LogprobForward p) {
  __shared__ Softmax sums[kMaxWaves];
  __shared__ float lane_best[kTop ? kMaxWaves : 1][64];
  __shared__ float notes[kTop ? kMaxWaves : 1][kNotes][64];
  __shared__ Found found;
  const int lane = lane_id(), wave = uniform(static_cast<int>(threadIdx.x / 64)), waves = blockDim.x / 64;
  const int row = uniform(static_cast<int>(blockIdx.x / p.parts)), part = uniform(static_cast<int>(blockIdx.x % p.parts));
  const float c2 = p.scale * kLog2e;
  const int64_t token = p.logprob ? p.tokens[row] : -1;
  if (kTop && threadIdx.x == 0) found.count = 0;
  Softmax a{kLowest, 0.f, 0.f};
  const int64_t batches = static_cast<int64_t>(p.batches_per_member) * p.members;
  const int first = static_cast<int>(batches * part / p.parts), end = static_cast<int>(batches * (part + 1) / p.parts);
  // batches of this wave that share a note
  const int per_note = ((end - first + waves - 1) / waves + kNotes - 1) / kNotes;
  float best = -INFINITY, note = -INFINITY;
  int turn = 0, at_note = 0;
  for (int b = first + wave; b < end; b += waves) {
    const Batch<T> batch = batch_at<T>(p, row, b);
    const float here = take_batch<T, kNt>(batch.p, batch.left, c2, a);
    if constexpr (kTop) {
      best = fmaxf(best, here);
      note = fmaxf(note, here);
      notes[wave][at_note][lane] = note;
      if (++turn == per_note) {
        turn = 0;
        ++at_note;
        note = -INFINITY;
      }
    }
  }
  // the token's logit, before what follows needs it
  float of_token = 0.f;
  if (wave == 0 && token >= 0 && token < p.vocab) of_token = logit_of<T>(p, row, token);
  a = join_lanes(a, c2);
  TopList t;
  top_clear(t);
  if (kTop || waves > 1) {
    if (lane == 0) sums[wave] = a;
    if constexpr (kTop) lane_best[wave][lane] = best;
    __syncthreads();
    if constexpr (kTop) {
      for (int w = 0; w < waves; ++w) best = fmaxf(best, lane_best[w][lane]);
      const float bound = bound_of_lanes(best, p.top_k);
      if (bound != -INFINITY) {
        turn = at_note = 0;
        for (int b = first + wave; b < end; b += waves) {
          const bool near = notes[wave][at_note][lane] >= bound;
          if (++turn == per_note) {
            turn = 0;
            ++at_note;
          }
          if (!__ballot(near) || *const_cast<volatile int *>(&found.count) > kMaxFound) continue;
          const Batch<T> batch = batch_at<T>(p, row, b);
          if (!near) continue;
          u32x4 raw[kDeep];
#pragma unroll
          for (int k = 0; k < kDeep; ++k) {
            const int c = (k * 64 + lane) * kRowVec<T>;
            raw[k] = row_load<T, true>(batch.p + c, batch.left - c, sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u);
          }
#pragma unroll
          for (int k = 0; k < kDeep; ++k)
#pragma unroll
            for (int e = 0; e < kRowVec<T>; ++e) {
              const float x = row_get<T>(raw[k], e);
              if (x >= bound) found_add(found, x, batch.id + (k * 64 + lane) * kRowVec<T> + e);
            }
        }
      }
      __syncthreads();
      if (wave != 0) return;
      if (bound != -INFINITY && found.count <= kMaxFound) {
        t = found_best(found, uniform(found.count), p.top_k);
      } else {
        for (int b = first; b < end; ++b) {
          const int w = (b - first) % waves, i = (b - first) / waves;
          const float noted = notes[w][i / per_note][lane];
          // ids grow from batch to batch: an equal value never beats a full list
          if (!__ballot(noted > t.last_value || t.last_id == kNoId)) continue;
          const Batch<T> batch = batch_at<T>(p, row, b);
          for (int e = 0; e < kBatch<T> / 64; ++e) {
            const int c = e * 64 + lane;
            top_offer(t, c < batch.left, element_at(batch, c), batch.id + c, p.top_k);
          }
        }
      }
    }
    if (wave != 0) return;
    a = lane < waves ? sums[lane] : Softmax{kLowest, 0.f, 0.f};
    a = join_lanes(a, c2);
  }
  if (p.parts == 1) {
    finish_row<kTop>(p, row, a, t, token, of_token);
    return;
  }
  // The workgroups of a row leave what they have; the one that arrives last joins it.  The words are
  // written past the L2 of the XCD (agent-scope stores), the writer waits for them, and only then counts
  // itself in; the last one reads them with agent-scope loads behind its count.  A release of the whole
  // L2 is not needed for them.
  const int64_t at = static_cast<int64_t>(row) * p.parts + part;
  float *mine = reinterpret_cast<float *>(p.part_sums + at);
  auto leave = [](auto *to, auto v) { __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  auto fetch = [](auto *from) { return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  if (lane < 3) leave(mine + lane, lane == 0 ? a.m : lane == 1 ? a.l : a.w);
  if constexpr (kTop) {
    if (lane < p.top_k) {
      leave(p.part_values + at * p.top_k + lane, t.value);
      leave(p.part_ids + at * p.top_k + lane, t.id);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  unsigned before = 0;
  if (lane == 0) before = __hip_atomic_fetch_add(p.arrived + 2 * row, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (uniform(before) != static_cast<unsigned>(p.parts - 1)) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  if (lane == 0) leave(p.arrived + 2 * row, 0u);
  a = {kLowest, 0.f, 0.f};
  if (lane < p.parts) {
    float *theirs = reinterpret_cast<float *>(p.part_sums + static_cast<int64_t>(row) * p.parts + lane);
    a = {fetch(theirs), fetch(theirs + 1), fetch(theirs + 2)};
  }
  if constexpr (kTop) {
    // the same bound over the parts' lists, all of them in registers
    constexpr int kHeld = kMaxParts * kMaxTop / 64;
    const int64_t lists = static_cast<int64_t>(row) * p.parts * p.top_k;
    const int n = p.parts * p.top_k;
    float v[kHeld];
    int id[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      const int i = k * 64 + lane;
      v[k] = -INFINITY;
      id[k] = kNoId;
      if (i < n) {
        v[k] = fetch(p.part_values + lists + i);
        id[k] = fetch(p.part_ids + lists + i);
      }
    }
    best = -INFINITY;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) best = fmaxf(best, v[k]);
    const float bound = bound_of_lanes(best, p.top_k);
    if (lane == 0) found.count = 0;
    __builtin_amdgcn_wave_barrier();
    if (bound != -INFINITY) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (v[k] >= bound) found_add(found, v[k], id[k]);
    }
    __builtin_amdgcn_wave_barrier();
    const int all = uniform(*const_cast<volatile int *>(&found.count));
    if (bound != -INFINITY && all <= kMaxFound) {
      t = found_best(found, all, p.top_k);
    } else {
      top_clear(t);
#pragma unroll 1
      for (int k = 0; k < kHeld; ++k) {
        const int i = k * 64 + lane;
        const float value = i < n ? fetch(p.part_values + lists + i) : -INFINITY;
        const int name = i < n ? fetch(p.part_ids + lists + i) : kNoId;
        top_offer(t, name != kNoId, value, name, p.top_k);
      }
    }
  }
  a = join_lanes(a, c2);
  finish_row<kTop>(p, row, a, t, token, of_token);
}

struct LogprobBackward {
  int rows, vocab, shard, members;
  int64_t step, ld, grad_ld;
  float scale;
  const char *logits;
  const int64_t *tokens;
  const float *lse, *entropy, *grad_logprob, *grad_entropy, *grad_lse;
  char *grad_logits;
  int chunks;   // workgroups per row of a member
};

// Bound by memory: without its arithmetic the kernel takes as long (4096 x 131072 bf16, by process 354
// or 382 us; 361 or 390 without arithmetic and 4 vectors per lane).  Eight vectors of a lane in flight:
// 391 us against 397 with four; stores past the caches' allocation on top: 382.
constexpr int kGradLanes = 256, kGradDeep = 8;
template <typename T>
constexpr int kGradChunk = kGradLanes * kRowVec<T> * kGradDeep;

template <typename T, bool kNt>
__global__ void __launch_bounds__(kGradLanes) logprob_grad_kernel(LogprobBackward p) {
  constexpr int V = kRowVec<T>;
  const uint64_t b = static_cast<uint64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
  const int chunk = uniform(static_cast<int>(b % p.chunks));
  const int64_t line = uniform(static_cast<unsigned long>(b / p.chunks));
  const int row = static_cast<int>(line / p.members), member = static_cast<int>(line % p.members);
  if (row >= p.rows) return;
  const int at = chunk * kGradChunk<T>;
  const int64_t id = static_cast<int64_t>(member) * p.shard + at;
  int left = p.shard - at;
  if (id + left > p.vocab) left = id < p.vocab ? static_cast<int>(p.vocab - id) : 0;
  if (left <= 0) return;
  const T *x = reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + at;
  T *out = reinterpret_cast<T *>(p.grad_logits + member * p.step) + row * p.grad_ld + at;
  const int lane = threadIdx.x;
  u32x4 raw[kGradDeep];
#pragma unroll
  for (int k = 0; k < kGradDeep; ++k) {
    const int c = (k * kGradLanes + lane) * V;
    raw[k] = row_load<T, true>(x + c, left - c);
  }
  // A row without any logit above minus infinity has no probabilities: 0 throughout, as against an
  // infinite normaliser.
  float lse = p.lse[row];
  if (lse == -INFINITY) lse = INFINITY;
  const int64_t token = p.tokens ? p.tokens[row] : -1;
  if (token >= p.vocab && chunk == 0 && member == 0 && lane == 0) status_raise(kStatusBadArgument);
  const float of_token = p.grad_logprob && token >= 0 && token < p.vocab ? p.scale * p.grad_logprob[row] : 0.f;
  const float of_entropy = p.grad_entropy ? p.scale * p.grad_entropy[row] : 0.f;
  const float of_lse = p.grad_lse ? p.scale * p.grad_lse[row] : 0.f;
  const float flat = of_lse - of_token - (p.grad_entropy ? of_entropy * p.entropy[row] : 0.f);
  const int64_t hit = token - id;
#pragma unroll
  for (int k = 0; k < kGradDeep; ++k) {
    const int c = (k * kGradLanes + lane) * V;
    float d[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float lp = fmaf(row_get<T>(raw[k], e), p.scale, -lse);
      d[e] = exp2_of(lp * kLog2e) * fmaf(-of_entropy, fmaxf(lp, kFarBelow), flat);
      if (c + e == hit) d[e] += of_token;
    }
    row_store<T, true, kNt>(out + c, left - c, row_pack<T>(d));
  }
}

// ---- host side ------------------------------------------------------------------------------------

size_t type_size(int dtype) { return dtype == RSM_FLOAT ? 4 : dtype == RSM_BF16 ? 2 : 0; }

struct LogprobShape {
  size_t shard, ld;
  rsm::Members team;
};

template <typename A>
bool shape_of(const A &a, const char *call, LogprobShape *out) {
  const std::string who = std::string(call) + ": ";
  auto refuse = [&](const char *why) {
    rsm::fail(who + why);
    return false;
  };
  LogprobShape s;
  if (!type_size(a.dtype)) return refuse("dtype must be RSM_FLOAT or RSM_BF16");
  if (a.vocab < 1 || a.vocab > 0x3fffffffull) return refuse("vocab must be in [1, 2^30)");
  if (a.rows >= 1u << 22) return refuse("rows must be below 2^22");
  if (!(a.scale > 0.f) || !std::isfinite(a.scale)) return refuse("scale must be a positive number");
  if (!rsm::members_of(a.team, call, &s.team)) return false;
  s.shard = a.shard ? a.shard : (a.vocab + s.team.size - 1) / s.team.size;
  if (s.shard > 0x3fffffffull || s.shard * s.team.size < a.vocab) return refuse("the members' shards do not cover the vocabulary");
  s.ld = a.logits_ld ? a.logits_ld : s.shard;
  if (s.ld < s.shard && s.ld < a.vocab) return refuse("a row stride is shorter than a row");
  if (s.ld > (~size_t{0} >> 24) / (a.rows + 1)) return refuse("a row stride is too long");
  *out = s;
  return true;
}

// The elements of a member's row that a call touches (the first member has the most).
size_t width_of(const LogprobShape &s, size_t vocab) { return s.shard < vocab ? s.shard : vocab; }

// How a row is cut: batches per member, workgroups per row and waves per workgroup.
struct LogprobPlan {
  int batches, parts, waves;
  size_t work_bytes;
};

LogprobPlan plan_of(const LogprobShape &s, int dtype, size_t rows, size_t vocab, int top_k) {
  LogprobPlan g{};
  const int batch = dtype == RSM_BF16 ? kBatch<__hip_bfloat16> : kBatch<float>;
  g.batches = static_cast<int>((width_of(s, vocab) + batch - 1) / batch);
  const int64_t all = static_cast<int64_t>(g.batches) * s.team.size;
  g.parts = 1;
  // Few rows: several workgroups to a row, so that the chip has some 512 to run, each with a batch for
  // each of its waves.  More and smaller ones lose more in the joining than they win (one row of 128000
  // bf16 with 20 alternatives: 8 workgroups of 8 waves 14.7 us, 16 of 4 15.3, 32 of 2 18.1, 64 of 1 24).
  if (rows && rows < 256) {
    int64_t parts = 512 / static_cast<int64_t>(rows);
    const int64_t most = (all + kMaxWaves - 1) / kMaxWaves;
    if (parts > most) parts = most;
    if (parts > kMaxParts) parts = kMaxParts;
    g.parts = parts < 1 ? 1 : static_cast<int>(parts);
  }
  const int64_t mine = (all + g.parts - 1) / g.parts;
  g.waves = mine < kMaxWaves ? static_cast<int>(mine) : kMaxWaves;
  if (g.parts > 1) g.work_bytes = rows * g.parts * (sizeof(float4) + static_cast<size_t>(top_k) * 8);
  return g;
}

const char *moved(const void *p, int64_t bytes) { return p ? static_cast<const char *>(p) + bytes : nullptr; }
char *moved(void *p, int64_t bytes) { return p ? static_cast<char *>(p) + bytes : nullptr; }
template <typename T>
const T *moved_as(const void *p, int64_t bytes) {
  return reinterpret_cast<const T *>(moved(p, bytes));
}

template <typename T>
void launch_forward(const LogprobForward &p, dim3 grid, dim3 block, hipStream_t st, bool once) {
  if (p.top_k) {
    if (once) hipLaunchKernelGGL((logprob_kernel<T, true, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((logprob_kernel<T, true, false>), grid, block, 0, st, p);
  } else {
    if (once) hipLaunchKernelGGL((logprob_kernel<T, false, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((logprob_kernel<T, false, false>), grid, block, 0, st, p);
  }
}

template <typename T>
void launch_backward(const LogprobBackward &p, dim3 grid, hipStream_t st, bool large) {
  if (large) hipLaunchKernelGGL((logprob_grad_kernel<T, true>), grid, dim3(kGradLanes), 0, st, p);
  else hipLaunchKernelGGL((logprob_grad_kernel<T, false>), grid, dim3(kGradLanes), 0, st, p);
}

bool top_in_range(const char *call, int top_k, size_t vocab) {
  if (top_k >= 0 && top_k <= kMaxTop && static_cast<size_t>(top_k) <= vocab) return true;
  rsm::fail(std::string(call) + ": top_k must be in [0, 32] and at most vocab");
  return false;
}

}  // namespace

extern "C" {

int rsm_logprob_work_bytes(const rsm_logprob_args_t *args, size_t *bytes) {
  RSM_ENTRY;
  const char *call = "logprob_work_bytes";
  if (!args || !bytes) return rsm::fail("logprob_work_bytes: an argument is NULL");
  LogprobShape s;
  if (!top_in_range(call, args->top_k, args->vocab) || !shape_of(*args, call, &s)) return -1;
  *bytes = plan_of(s, args->dtype, args->rows, args->vocab, args->top_k).work_bytes;
  return 0;
}

int rsm_logprob_to_all(const rsm_logprob_args_t *args, void *stream) {
  RSM_ENTRY;
  const char *call = "logprob_to_all";
  if (!args) return rsm::fail("logprob_to_all: arguments are NULL");
  const rsm_logprob_args_t &a = *args;
  LogprobShape s;
  if (!a.logits) return rsm::fail("logprob_to_all: logits must be given");
  if (a.logprob && !a.tokens) return rsm::fail("logprob_to_all: logprob without tokens");
  if (!a.logprob && !a.entropy && !a.lse && !a.top_ids && !a.top_logprobs) return rsm::fail("logprob_to_all: no result is asked for");
  if ((a.top_ids || a.top_logprobs) != (a.top_k > 0)) return rsm::fail("logprob_to_all: top_k and the arrays for the alternatives do not go together");
  if (!top_in_range(call, a.top_k, a.vocab) || !shape_of(a, call, &s)) return -1;
  const LogprobPlan g = plan_of(s, a.dtype, a.rows, a.vocab, a.top_k);
  if (g.parts > 1 && (!a.work || !a.pSync)) return rsm::fail("logprob_to_all: work (rsm_logprob_work_bytes) and pSync must be given for so few rows");
  if (a.rows == 0) return 0;
  const size_t size = type_size(a.dtype);
  rsm::Operands o(call);
  o.matrix(a.logits, "logits", a.rows, width_of(s, a.vocab), s.ld, size, false);
  o.add(a.tokens, "tokens", a.rows * 8, false);
  o.add(a.logprob, "logprob", a.rows * 4, true);
  o.add(a.entropy, "entropy", a.rows * 4, true);
  o.add(a.lse, "lse", a.rows * 4, true);
  o.add(a.top_ids, "top_ids", a.rows * a.top_k * 4, true);
  o.add(a.top_logprobs, "top_logprobs", a.rows * a.top_k * 4, true);
  if (g.parts > 1) {
    o.add(a.work, "work (rsm_logprob_work_bytes)", g.work_bytes, true);
    o.add(a.pSync, "pSync (ROC_SHMEM_REDUCE_SYNC_SIZE longs)", ROC_SHMEM_REDUCE_SYNC_SIZE * sizeof(long), true);
  }
  if (!o.ok()) return -1;
  LogprobForward p{};
  p.rows = static_cast<int>(a.rows);
  p.vocab = static_cast<int>(a.vocab);
  p.shard = static_cast<int>(s.shard);
  p.members = s.team.size;
  p.top_k = a.top_k;
  p.step = s.team.step;
  p.ld = static_cast<int64_t>(s.ld);
  p.scale = a.scale;
  p.logits = moved(a.logits, s.team.first);
  p.tokens = moved_as<int64_t>(a.tokens, s.team.first);
  p.logprob = moved(a.logprob, s.team.first);
  p.entropy = moved(a.entropy, s.team.first);
  p.lse = moved(a.lse, s.team.first);
  p.top_ids = moved(a.top_ids, s.team.first);
  p.top_logprobs = moved(a.top_logprobs, s.team.first);
  p.batches_per_member = g.batches;
  p.parts = g.parts;
  if (g.parts > 1) {
    const size_t n = a.rows * g.parts;
    char *work = moved(a.work, s.team.first);
    p.part_sums = reinterpret_cast<float4 *>(work);
    p.part_values = reinterpret_cast<float *>(work + n * sizeof(float4));
    p.part_ids = reinterpret_cast<int *>(p.part_values + n * a.top_k);
    p.arrived = reinterpret_cast<unsigned *>(moved(a.pSync, s.team.first));
  }
  const dim3 grid(static_cast<unsigned>(a.rows * g.parts)), block(static_cast<unsigned>(g.waves * 64));
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Logits that the Infinity Cache could not hold anyway are read past it: 4096 x 131072 bf16 without
  // alternatives 168 us against 186; smaller ones may still lie there from the product that made them.
  const bool once = a.rows * a.vocab * size > rsm::kInfinityCacheBytes;
  if (a.dtype == RSM_BF16) launch_forward<__hip_bfloat16>(p, grid, block, st, once);
  else launch_forward<float>(p, grid, block, st, once);
  return rsm::after_launch(call);
}

int rsm_logprob_to_all_grad(const rsm_logprob_grad_args_t *args, void *stream) {
  RSM_ENTRY;
  const char *call = "logprob_to_all_grad";
  if (!args) return rsm::fail("logprob_to_all_grad: arguments are NULL");
  const rsm_logprob_grad_args_t &a = *args;
  LogprobShape s;
  if (!a.logits || !a.lse || !a.grad_logits) return rsm::fail("logprob_to_all_grad: logits, lse and grad_logits must be given");
  if (!a.grad_logprob && !a.grad_entropy && !a.grad_lse) return rsm::fail("logprob_to_all_grad: no gradient is given");
  if (a.grad_logprob && !a.tokens) return rsm::fail("logprob_to_all_grad: grad_logprob without tokens");
  if (a.grad_entropy && !a.entropy) return rsm::fail("logprob_to_all_grad: grad_entropy without entropy");
  if (!shape_of(a, call, &s)) return -1;
  const size_t grad_ld = a.grad_ld ? a.grad_ld : s.shard, width = width_of(s, a.vocab);
  if (grad_ld < width) return rsm::fail("logprob_to_all_grad: a row stride is shorter than a row");
  if (grad_ld > (~size_t{0} >> 24) / (a.rows + 1)) return rsm::fail("logprob_to_all_grad: a row stride is too long");
  if (a.rows == 0) return 0;
  const size_t size = type_size(a.dtype);
  rsm::Operands o(call);
  o.matrix(a.logits, "logits", a.rows, width, s.ld, size, false);
  o.add(a.tokens, "tokens", a.rows * 8, false);
  o.add(a.lse, "lse", a.rows * 4, false);
  o.add(a.entropy, "entropy", a.rows * 4, false);
  o.add(a.grad_logprob, "grad_logprob", a.rows * 4, false);
  o.add(a.grad_entropy, "grad_entropy", a.rows * 4, false);
  o.add(a.grad_lse, "grad_lse", a.rows * 4, false);
  o.matrix(a.grad_logits, "grad_logits", a.rows, width, grad_ld, size, true);
  if (grad_ld == s.ld) o.or_same_as(a.logits);
  if (!o.ok()) return -1;
  LogprobBackward p{};
  p.rows = static_cast<int>(a.rows);
  p.vocab = static_cast<int>(a.vocab);
  p.shard = static_cast<int>(s.shard);
  p.members = s.team.size;
  p.step = s.team.step;
  p.ld = static_cast<int64_t>(s.ld);
  p.grad_ld = static_cast<int64_t>(grad_ld);
  p.scale = a.scale;
  p.logits = moved(a.logits, s.team.first);
  p.tokens = moved_as<int64_t>(a.tokens, s.team.first);
  p.lse = moved_as<float>(a.lse, s.team.first);
  p.entropy = moved_as<float>(a.entropy, s.team.first);
  p.grad_logprob = moved_as<float>(a.grad_logprob, s.team.first);
  p.grad_entropy = moved_as<float>(a.grad_entropy, s.team.first);
  p.grad_lse = moved_as<float>(a.grad_lse, s.team.first);
  p.grad_logits = moved(a.grad_logits, s.team.first);
  const size_t per = a.dtype == RSM_BF16 ? kGradChunk<__hip_bfloat16> : kGradChunk<float>;
  p.chunks = static_cast<int>((width + per - 1) / per);
  const size_t wgs = a.rows * p.members * static_cast<size_t>(p.chunks);
  const size_t x = wgs < 0x800000 ? wgs : 0x800000, y = (wgs + x - 1) / x;
  if (y > 65535) return rsm::fail("logprob_to_all_grad: too many rows for one launch");
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool large = 2 * a.rows * a.vocab * size > rsm::kInfinityCacheBytes;
  if (a.dtype == RSM_BF16) launch_backward<__hip_bfloat16>(p, grid, st, large);
  else launch_backward<float>(p, grid, st, large);
  return rsm::after_launch(call);
}

}  // extern "C"
