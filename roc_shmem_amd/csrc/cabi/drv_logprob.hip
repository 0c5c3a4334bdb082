// C ABI: log probabilities over a vocabulary that is split over the members of a team, and their
// gradient (rsm_logprob_to_all, rsm_logprob_to_all_grad; no counterpart in the reference).
//
// With x a row's logits over all members, y = c x and m = max y:
//   l = sum exp(y - m)          lse = m + ln l
//   logprob = y[token] - lse    entropy = ln l - sum exp(y - m) (y - m) / l
//   top: the k largest x, equal ones by ascending id, with their log probabilities
// and backwards, with p = exp(y - lse) = exp(c (x - max x) - ln l):
//   dx = c (g_logprob (1[token] - p) + g_lse p - g_entropy p (ln p + entropy))
// The second form of p is the forward pass's own, good whatever the size of lse; the first, from lse as a
// float, has p off by 2^-24 |lse| of itself.
//
// The forward pass reads every logit once.  A lane keeps a running maximum m of its own x, and
// l = sum 2^((x - m) c2) and w = sum 2^((x - m) c2) (x - m) c2, c2 = c log2(e), against it; when m
// grows by d both shrink by 2^(-d c2).  Differences are taken before they are scaled, so rows whose
// logits are all at the type's lowest value come out as any other row of equal logits.  A logit at
// minus infinity has probability 0 and adds nothing to the entropy; m starts at the lowest finite
// value, not at minus infinity, so that such logits never meet an infinite m.
#include <cfloat>
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

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }

constexpr int kMaxWaves = 8, kMaxParts = 16;

struct LogprobForward {
  int rows, vocab, shard, members, top_k;
  int64_t step, ld;
  float scale;
  const char *logits;
  const int64_t *tokens;
  char *logprob, *entropy, *lse, *largest, *log_sum, *top_ids, *top_logprobs;
  // A row is cut into batches of kBatch elements, 64 lanes x kDeep vectors, in ascending order of ids;
  // workgroup q of `parts` takes its share of them in order.  Either every member's part is cut for
  // itself (batches_per_member), or, where that would leave the last batches mostly empty (kPacked),
  // the parts' vectors (vecs of them to a member) are numbered through and 256 of them make a batch.
  int batches, batches_per_member, parts;
  unsigned vecs, per_vecs;   // per_vecs: 2^32 / vecs, rounded up (exact for as few vectors); 0: vecs is 1
  float4 *part_sums;     // [rows][parts]: m, l, w
  uint64_t *part_keys;   // [rows][parts][top_k]
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

// Minus infinity in every element of a 32-bit word.
template <typename T>
constexpr uint32_t kMinusInf = sizeof(T) == 4 ? 0xff800000u : 0xff80ff80u;

// Where a vector of a lane lies in a row: its first element, how many there are from it on (perhaps
// none), and the first one's id.
template <typename T>
struct Place {
  const T *p;
  int left, id;
};

// Elements of member m's part from element `at` on.
__device__ __forceinline__ int elements_left(const LogprobForward &p, int member, int at) {
  const int64_t id = static_cast<int64_t>(member) * p.shard + at;
  const int64_t rest = p.vocab - id;
  if (rest <= 0) return 0;
  return rest < p.shard - at ? static_cast<int>(rest) : p.shard - at;
}

// Vector `c / kRowVec` of batch b, with `c` the element's number within the batch.
template <typename T, bool kPacked>
struct Batch {
  const LogprobForward &p;
  int row, b;
  const T *part;      // not packed: the batch's first element, and what is left from there on
  int left, id;
  __device__ __forceinline__ Batch(const LogprobForward &p_, int row_, int b_) : p(p_), row(row_), b(b_) {
    if constexpr (!kPacked) {
      const int member = uniform(b / p.batches_per_member);
      const int at = (b - member * p.batches_per_member) * kBatch<T>;
      left = elements_left(p, member, at);
      id = static_cast<int>(static_cast<int64_t>(member) * p.shard + at);
      part = reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + at;
    }
  }
  __device__ __forceinline__ Place<T> at(int c) const {
    if constexpr (kPacked) {
      const unsigned j = static_cast<unsigned>(b * kBatch<T> + c) / kRowVec<T>;
      const int member = static_cast<int>(p.per_vecs ? __umulhi(j, p.per_vecs) : j);
      const int off = static_cast<int>(j - member * p.vecs) * kRowVec<T> + c % kRowVec<T>;
      const int rest = member < p.members ? elements_left(p, member, off) : 0;
      // beyond the last member's part, where nothing is left, the id would not fit an int
      const unsigned id = static_cast<unsigned>(member) * static_cast<unsigned>(p.shard) + static_cast<unsigned>(off);
      return {reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + off, rest, static_cast<int>(id)};
    } else {
      return {part + c, left - c, id + c};
    }
  }
};

// The same for a batch of each lane's own.
template <typename T, bool kPacked>
__device__ __forceinline__ Place<T> place_in(const LogprobForward &p, int row, int b, int c) {
  if constexpr (kPacked) {
    return Batch<T, true>(p, row, b).at(c);
  } else {
    const int member = static_cast<int>(static_cast<unsigned>(b) / static_cast<unsigned>(p.batches_per_member));
    const int at = (b - member * p.batches_per_member) * kBatch<T> + c;
    return {reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + at, elements_left(p, member, at),
            static_cast<int>(static_cast<int64_t>(member) * p.shard + at)};
  }
}

template <typename T, bool kNt, bool kPacked>
__device__ __forceinline__ void load_batch(const Batch<T, kPacked> &batch, u32x4 (&raw)[kDeep]) {
#pragma unroll
  for (int k = 0; k < kDeep; ++k) {
    const Place<T> v = batch.at((k * 64 + lane_id()) * kRowVec<T>);
    raw[k] = row_load<T, true, kNt>(v.p, v.left, kMinusInf<T>);
  }
}

// One batch of a wave.  Returns the largest of this lane's elements.
template <typename T>
__device__ __forceinline__ float take_batch(const u32x4 (&raw)[kDeep], float c2, Softmax &a) {
  constexpr int V = kRowVec<T>;
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
// caches), their elements above it are gathered in LDS, and one wave ranks them.  The price per logit
// is nothing but the maximum that the softmax needs anyway.  Where fewer than k groups have a number
// above minus infinity, all such numbers are gathered, and the lowest ids at minus infinity follow
// them.  Rows of which a wave finds more than kRoom elements (many equal values) are gone through
// once more in ascending order of ids, batch by batch, into a sorted list.
//
// An element is a 64-bit key: its value, ordered as an unsigned number, above its id counted down, so
// that the larger of two keys is the larger value or, of equal ones, the lower id; 0 is no element.
typedef uint64_t Key;
constexpr int kRoom = 64, kNotes = 16;

__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of_order(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ Key key_of(float v, int id) {
  return static_cast<Key>(order_of(v + 0.f)) << 32 | ~static_cast<uint32_t>(id);   // -0 equals 0
}
__device__ __forceinline__ float value_of(Key k) { return value_of_order(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int id_of(Key k) { return static_cast<int>(~static_cast<uint32_t>(k)); }
__device__ __forceinline__ Key lane_key(Key k, int lane) {
  return static_cast<Key>(__builtin_amdgcn_readlane(static_cast<uint32_t>(k >> 32), lane)) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(k), lane));
}

// The order of a value, in 16 bits and not above it, that the k largest of the lanes' orders reach.
__device__ __forceinline__ uint32_t bound_of_lanes(uint32_t order, int k) {
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t with = bound | 1u << bit;
    if (__popcll(__ballot(order >= with)) >= k) bound = with;
  }
  return bound;
}
constexpr uint32_t kOrderOfMinusInf = 0x007fffffu;   // what is not above it bounds nothing

// A wave's best elements in a sorted list: lane r holds the one of rank r.
struct TopList {
  Key key;
  Key last;   // the element of rank top_k - 1, the same in every lane: what another must beat
};

// Every lane offers one element (0: none).
__device__ __forceinline__ void top_offer(TopList &t, Key offered, int top_k) {
  uint64_t mask = __ballot(offered > t.last);
  while (mask) {
    const Key key = lane_key(offered, __builtin_ctzll(mask));
    mask &= mask - 1;
    if (key <= t.last) continue;
    const int rank = __popcll(__ballot(t.key > key)), lane = lane_id();
    const Key up = from_lower_lane(t.key);
    t.key = lane > rank ? up : lane == rank ? key : t.key;
    t.last = lane_key(t.key, top_k - 1);
  }
}

// What a workgroup's waves share, in LDS: `waves` of each array.
struct Shared {
  float (*notes)[kNotes][64];   // [wave][note][lane]: the largest element of a batch, or of several
  float (*best)[64];            // [wave][lane]: the largest element of all
  Key (*found)[kRoom];          // [wave]: the elements it gathered
  Key *all;                     // [64]
  Softmax *sums;                // [wave]
  int *count;                   // [wave]: how many it gathered, kRoom + 1 or more: too many
};
__host__ __device__ constexpr size_t shared_bytes(int waves, bool top) {
  return waves * (sizeof(Softmax) + (top ? (kNotes + 1) * 64 * sizeof(float) + kRoom * sizeof(Key) + sizeof(int) : 0)) +
         (top ? 64 * sizeof(Key) : 0);
}
__device__ __forceinline__ Shared shared_of(char *base, int waves, bool top) {
  Shared s{};
  if (top) {
    s.found = reinterpret_cast<Key(*)[kRoom]>(base);
    s.all = reinterpret_cast<Key *>(s.found + waves);
    s.notes = reinterpret_cast<float(*)[kNotes][64]>(s.all + 64);
    s.best = reinterpret_cast<float(*)[64]>(s.notes + waves);
    s.count = reinterpret_cast<int *>(s.best + waves);
    base = reinterpret_cast<char *>(s.count + waves);
  }
  s.sums = reinterpret_cast<Softmax *>(base);
  return s;
}

// Appends the lanes' elements (hit: there is one) to a wave's; `n` counts on beyond the room.
__device__ __forceinline__ void found_add(Key *found, int &n, bool hit, Key key) {
  const uint64_t mask = __ballot(hit);
  if (mask == 0) return;
  const int at = n + rank_in_mask(mask);
  if (hit && at < kRoom) found[at] = key;
  n += __popcll(mask);
}

// What `waves` waves found, at most kRoom each, sorted by one wave.
__device__ __forceinline__ TopList found_best(const Shared &s, int waves, int top_k) {
  TopList t{0, 0};
  const int lane = lane_id();
  int n = 0;
  Key mine = 0;
  for (int w = 0; w < waves; ++w) {
    const int c = uniform(s.count[w]);
    if (lane >= n && lane < n + c) mine = s.found[w][lane - n];
    n += c;
  }
  if (n > 64) {
    for (int w = 0; w < waves; ++w) top_offer(t, lane < s.count[w] ? s.found[w][lane] : 0, top_k);
    return t;
  }
  s.all[lane] = mine;
  __builtin_amdgcn_wave_barrier();
  int rank = 0;
  for (int i = 0; i < n; i += 8) {   // beyond n the keys are 0 and beat nobody
#pragma unroll
    for (int j = 0; j < 8; ++j) rank += s.all[i + j] > mine;
  }
  if (lane >= n) rank = lane;
  // every lane sends its element to the lane of its rank
  const uint32_t high = __builtin_amdgcn_ds_permute(rank * 4, static_cast<int>(mine >> 32));
  const uint32_t low = __builtin_amdgcn_ds_permute(rank * 4, static_cast<int>(mine));
  t.key = static_cast<Key>(high) << 32 | low;
  t.last = lane_key(t.key, top_k - 1);
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
    if (p.largest) reinterpret_cast<float *>(p.largest + m * p.step)[row] = empty ? -INFINITY : a.m;
    if (p.log_sum) reinterpret_cast<float *>(p.log_sum + m * p.step)[row] = empty ? -INFINITY : log_l;
  }
  if constexpr (kTop) {
    if (lane < p.top_k) {
      const int64_t at = static_cast<int64_t>(row) * p.top_k + lane;
      // a row of fewer than k numbers (the others NaN) has no more to name
      const bool none = t.key == 0;
      const float lp = none ? NAN : empty ? -INFINITY : fmaf(p.scale, value_of(t.key) - a.m, -log_l);
      for (int m = 0; m < p.members; ++m) {
        if (p.top_ids) reinterpret_cast<int *>(p.top_ids + m * p.step)[at] = none ? -1 : id_of(t.key);
        if (p.top_logprobs) reinterpret_cast<float *>(p.top_logprobs + m * p.step)[at] = lp;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ float element_at(const Place<T> &v) {
  if (v.left <= 0) return -INFINITY;
  if constexpr (sizeof(T) == 4) return *v.p;
  else return bf16_bits_to_float(*reinterpret_cast<const uint16_t *>(v.p));
}

// Without alternatives the stream of logits bounds it: 4096 x 131072 bf16 over 8 members 164 us, 6.5 TB/s, as
// for half as many float ones; with 8 of them 185.  One row of 128000 over 8 members with 20 takes 10 us, a chain
// of phases: 2 to stream, 3 to bound and rank, 3 to join the workgroups, 1 to write.
//
// 64 vector registers at most, so that a compute unit holds four workgroups: while some rank their
// row's alternatives the others stream.  kSingle: no wave has more than one batch of alternatives to look
// at, which then stays in its registers (4096 x 16000 bf16, 8 alternatives: 42 us against 47; one row of 128000
// over 8 members, 20 of them: 10.6 against 11.2).
template <typename T, bool kTop, bool kNt, bool kPacked, bool kSingle>
__global__ void __launch_bounds__(kMaxWaves * 64, 8) logprob_kernel(LogprobForward p) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = lane_id(), wave = uniform(static_cast<int>(threadIdx.x / 64)), waves = blockDim.x / 64;
  const Shared sh = shared_of(lds, waves, kTop);
  const int row = uniform(static_cast<int>(blockIdx.x / p.parts)), part = uniform(static_cast<int>(blockIdx.x % p.parts));
  const float c2 = p.scale * kLog2e;
  const int64_t token = p.logprob ? p.tokens[row] : -1;
  Softmax a{kLowest, 0.f, 0.f};
  const int first = static_cast<int>(static_cast<int64_t>(p.batches) * part / p.parts);
  const int end = static_cast<int>(static_cast<int64_t>(p.batches) * (part + 1) / p.parts);
  // batches of this wave that share a note
  const int per_note = ((end - first + waves - 1) / waves + kNotes - 1) / kNotes;
  float best = -INFINITY, note = -INFINITY;
  int turn = 0, at_note = 0;
  u32x4 kept[kDeep];   // kSingle: the wave's only batch
  if constexpr (kSingle) {
    if (first + wave < end) {
      load_batch<T, kNt>(Batch<T, kPacked>(p, row, first + wave), kept);
      best = take_batch<T>(kept, c2, a);
    }
  }
  for (int b = first + wave; !kSingle && b < end; b += waves) {
    u32x4 raw[kDeep];
    load_batch<T, kNt>(Batch<T, kPacked>(p, row, b), raw);
    const float here = take_batch<T>(raw, c2, a);
    if constexpr (kTop) {
      best = fmaxf(best, here);
      note = fmaxf(note, here);
      sh.notes[wave][at_note][lane] = note;
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
  TopList t{0, 0};
  if (kTop || waves > 1) {
    if (lane == 0) sh.sums[wave] = a;
    if constexpr (kTop) sh.best[wave][lane] = best;
    __syncthreads();
    if constexpr (kTop) {
      const float here = best;
      for (int w = 0; w < waves; ++w) best = fmaxf(best, sh.best[w][lane]);
      const uint32_t order = bound_of_lanes(order_of(best), p.top_k);
      const bool bounded = order > kOrderOfMinusInf;
      const float bound = bounded ? value_of_order(order) : kLowest;
      int n = 0;
      auto gather = [&](const u32x4 (&raw)[kDeep], const int (&id)[kDeep]) {
#pragma unroll
        for (int k = 0; k < kDeep; ++k)
#pragma unroll
          for (int e = 0; e < kRowVec<T>; ++e) {
            const float x = row_get<T>(raw[k], e);
            found_add(sh.found[wave], n, x >= bound, key_of(x, id[k] + e));
          }
      };
      if constexpr (kSingle) {
        if (__ballot(here >= bound)) {
          const Batch<T, kPacked> batch(p, row, first + wave);
          int id[kDeep];
#pragma unroll
          for (int k = 0; k < kDeep; ++k) id[k] = batch.at((k * 64 + lane) * kRowVec<T>).id;
          gather(kept, id);
        }
      } else {
        // What is near the bound, a lane's vectors of a batch each, is read by 64 lanes at a time, so that
        // the wave waits for memory once and not for every batch: lane r holds the r-th of them.
        int near_ones = 0, one = 0;
        auto look = [&] {
          u32x4 raw[kDeep];
          int id[kDeep];
#pragma unroll
          for (int k = 0; k < kDeep; ++k) {
            const Place<T> v = place_in<T, kPacked>(p, row, one >> 6, (k * 64 + (one & 63)) * kRowVec<T>);
            id[k] = v.id;
            raw[k] = row_load<T, true>(v.p, lane < near_ones ? v.left : 0, kMinusInf<T>);
          }
          gather(raw, id);
          near_ones = 0;
        };
        turn = at_note = 0;
        for (int b = first + wave; b < end && n <= kRoom; b += waves) {
          const uint64_t near = __ballot(sh.notes[wave][at_note][lane] >= bound);
          if (++turn == per_note) {
            turn = 0;
            ++at_note;
          }
          if (near == 0) continue;
          const int more = __popcll(near), below = rank_in_mask(near);
          if (near_ones + more > 64) look();
          // to the free lanes in order, the others' behind them
          const int to = near_ones + (near >> lane & 1 ? below : more + lane - below);
          const int sent = __builtin_amdgcn_ds_permute((to & 63) * 4, b << 6 | lane);
          if (lane >= near_ones && lane < near_ones + more) one = sent;
          near_ones += more;
        }
        if (near_ones > 0 && n <= kRoom) look();
      }
      if (lane == 0) sh.count[wave] = n;
      __syncthreads();
      if (wave != 0) return;
      const bool room = __ballot(lane < waves && sh.count[lane % waves] > kRoom) == 0;
      if (room) t = found_best(sh, waves, p.top_k);
      if (!room || t.last == 0) {
        // Ids grow from batch to batch: an equal value never beats a full list.  Behind all numbers
        // above minus infinity (room) only elements at minus infinity are missing.
        for (int b = first; b < end && !(room && t.last != 0); ++b) {
          const int w = (b - first) % waves, i = (b - first) / waves;
          const uint32_t noted = order_of((kSingle ? sh.best[w][lane] : sh.notes[w][i / per_note][lane]) + 0.f);
          if (!__ballot(noted > static_cast<uint32_t>(t.last >> 32))) continue;
          const Batch<T, kPacked> batch(p, row, b);
          for (int e = 0; e < kBatch<T> / 64; ++e) {
            const Place<T> v = batch.at(e * 64 + lane);
            const float x = element_at(v);
            top_offer(t, v.left > 0 && (room ? x == -INFINITY : x == x) ? key_of(x, v.id) : 0, p.top_k);
          }
        }
      }
    }
    if (wave != 0) return;
    a = lane < waves ? sh.sums[lane] : Softmax{kLowest, 0.f, 0.f};
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
      leave(p.part_keys + at * p.top_k + lane, t.key);
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
    uint64_t *lists = p.part_keys + static_cast<int64_t>(row) * p.parts * p.top_k;
    const int n = p.parts * p.top_k;
    Key held[kHeld], most = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
      held[k] = 0;
      if (k * 64 + lane < n) held[k] = fetch(lists + k * 64 + lane);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) most = held[k] > most ? held[k] : most;
    const uint32_t bound = bound_of_lanes(static_cast<uint32_t>(most >> 32), p.top_k);
    int count = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      found_add(sh.found[0], count, static_cast<uint32_t>(held[k] >> 32) >= bound && held[k] != 0, held[k]);
    if (count <= kRoom) {
      if (lane == 0) sh.count[0] = count;
      __builtin_amdgcn_wave_barrier();
      t = found_best(sh, 1, p.top_k);
    } else {
      t = {0, 0};
#pragma unroll
      for (int k = 0; k < kHeld; ++k) top_offer(t, held[k], p.top_k);
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
  const float *largest, *normaliser;   // of a row: ln p = scale (x - largest) - normaliser; largest null: 0
  const float *entropy, *grad_logprob, *grad_entropy, *grad_lse;
  char *grad_logits;
  // A line is one member's part of a row.  Either `chunks` workgroups take a line, or, where that would
  // leave them mostly idle (kPacked), the lines' vectors (vecs of them to a line) are numbered through.
  int chunks;
  unsigned vecs, per_vecs, per_members;   // per_*: 2^32 / *, rounded up (exact for what is divided); 0: * is 1
};

// Bound by memory: without its arithmetic the kernel takes as long (4096 x 131072 bf16, by process 354
// or 382 us; 361 or 390 without arithmetic and 4 vectors per lane).  Eight vectors of a lane in flight:
// 391 us against 397 with four; stores past the caches' allocation on top: 382.
constexpr int kGradLanes = 256, kGradDeep = 8;
template <typename T>
constexpr int kGradChunk = kGradLanes * kRowVec<T> * kGradDeep;

// What the gradient of a row's logits depends on.
struct RowGrads {
  float largest, normaliser, of_token, of_entropy, flat;
  int64_t token;
};
__device__ __forceinline__ RowGrads row_grads(const LogprobBackward &p, int row) {
  RowGrads r;
  r.largest = p.largest ? p.largest[row] : 0.f;
  r.normaliser = p.normaliser[row];
  // A row without any logit above minus infinity has no probabilities: they are 0 throughout, as against
  // an infinite normaliser, and what is left of its gradient is the token's own term.
  if (r.normaliser == -INFINITY) {
    r.largest = 0.f;
    r.normaliser = INFINITY;
  }
  r.token = p.tokens ? p.tokens[row] : -1;
  r.of_token = p.grad_logprob && r.token >= 0 && r.token < p.vocab ? p.scale * p.grad_logprob[row] : 0.f;
  r.of_entropy = p.grad_entropy ? p.scale * p.grad_entropy[row] : 0.f;
  r.flat = (p.grad_lse ? p.scale * p.grad_lse[row] : 0.f) - r.of_token - (p.grad_entropy ? r.of_entropy * p.entropy[row] : 0.f);
  return r;
}

// The gradient of a vector of logits whose first element has id `id`.
template <typename T>
__device__ __forceinline__ u32x4 grad_of(const LogprobBackward &p, const RowGrads &r, u32x4 raw, int64_t id) {
  const int64_t hit = r.token - id;
  float d[kRowVec<T>];
#pragma unroll
  for (int e = 0; e < kRowVec<T>; ++e) {
    const float lp = fmaf(row_get<T>(raw, e) - r.largest, p.scale, -r.normaliser);
    d[e] = exp2_of(lp * kLog2e) * fmaf(-r.of_entropy, fmaxf(lp, kFarBelow), r.flat);
    if (e == hit) d[e] += r.of_token;
  }
  return row_pack<T>(d);
}

// j / n for the small j of packed vectors and members; per_n: see LogprobBackward.
__device__ __forceinline__ int divided(unsigned j, unsigned per_n) { return static_cast<int>(per_n ? __umulhi(j, per_n) : j); }

template <typename T, bool kNt, bool kPacked>
__global__ void __launch_bounds__(kGradLanes) logprob_grad_kernel(LogprobBackward p) {
  constexpr int V = kRowVec<T>;
  const uint64_t b = static_cast<uint64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
  const int lane = threadIdx.x;
  u32x4 raw[kGradDeep];
  if constexpr (kPacked) {
    const uint64_t first = b * (kGradLanes * kGradDeep);
    const uint64_t line0 = uniform(static_cast<unsigned long>(first / p.vecs));
    const unsigned into = uniform(static_cast<uint32_t>(first % p.vecs));
    const int64_t row0 = uniform(static_cast<unsigned long>(line0 / p.members));
    const unsigned member0 = uniform(static_cast<uint32_t>(line0 % p.members));
    auto at = [&](int k, int64_t *row, int *off, int *member) {
      const unsigned j = into + k * kGradLanes + lane;
      const int line = divided(j, p.per_vecs);
      *off = static_cast<int>(j - line * p.vecs) * V;
      const unsigned q = member0 + line;
      const int down = divided(q, p.per_members);
      *member = static_cast<int>(q) - down * p.members;
      *row = row0 + down;
      const int64_t left = p.vocab - (static_cast<int64_t>(*member) * p.shard + *off);
      const int width = p.shard - *off;
      return *row >= p.rows || left <= 0 ? 0 : left < width ? static_cast<int>(left) : width;
    };
    int64_t row;
    int off, member;
#pragma unroll
    for (int k = 0; k < kGradDeep; ++k) {
      const int left = at(k, &row, &off, &member);
      raw[k] = row_load<T, true>(reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + off, left);
    }
#pragma unroll
    for (int k = 0; k < kGradDeep; ++k) {
      const int left = at(k, &row, &off, &member);
      if (left > 0) {
        const RowGrads r = row_grads(p, static_cast<int>(row));
        if (r.token >= p.vocab && member == 0 && off == 0) status_raise(kStatusBadArgument);
        row_store<T, true, kNt>(reinterpret_cast<T *>(p.grad_logits + member * p.step) + row * p.grad_ld + off, left,
                                grad_of<T>(p, r, raw[k], static_cast<int64_t>(member) * p.shard + off));
      }
    }
  } else {
    const int chunk = uniform(static_cast<int>(b % p.chunks));
    const int64_t line = uniform(static_cast<unsigned long>(b / p.chunks));
    const int row = static_cast<int>(line / p.members), member = static_cast<int>(line % p.members);
    if (row >= p.rows) return;
    const int at = chunk * kGradChunk<T>;
    const int64_t id = static_cast<int64_t>(member) * p.shard + at;
    const int64_t rest = p.vocab - id;
    const int left = rest <= 0 ? 0 : rest < p.shard - at ? static_cast<int>(rest) : p.shard - at;
    const T *x = reinterpret_cast<const T *>(p.logits + member * p.step) + row * p.ld + at;
    T *out = reinterpret_cast<T *>(p.grad_logits + member * p.step) + row * p.grad_ld + at;
#pragma unroll
    for (int k = 0; k < kGradDeep; ++k) {
      const int c = (k * kGradLanes + lane) * V;
      raw[k] = row_load<T, true>(x + c, left - c);
    }
    const RowGrads r = row_grads(p, row);
    if (r.token >= p.vocab && chunk == 0 && member == 0 && lane == 0) status_raise(kStatusBadArgument);
#pragma unroll
    for (int k = 0; k < kGradDeep; ++k) {
      const int c = (k * kGradLanes + lane) * V;
      row_store<T, true, kNt>(out + c, left - c, grad_of<T>(p, r, raw[k], id + c));
    }
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
  auto refuse = [&](const char *why) {
    rsm::fail(std::string(call) + ": " + why);
    return false;
  };
  LogprobShape s;
  if (!type_size(a.dtype)) return refuse("dtype must be RSM_FLOAT or RSM_BF16");
  if (a.vocab < 1 || a.vocab > 0x3fffffffull) return refuse("vocab must be in [1, 2^30)");
  if (a.rows >= 1u << 22) return refuse("rows must be below 2^22");
  if (!(a.scale >= FLT_MIN) || !std::isfinite(a.scale * kLog2e)) return refuse("scale must be a positive (normal) number below 2^127");
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
  int batches, batches_per_member, parts, waves;
  unsigned vecs;
  bool packed;
  size_t work_bytes;
};

LogprobPlan plan_of(const LogprobShape &s, int dtype, size_t rows, size_t vocab, int top_k) {
  LogprobPlan g{};
  const int vec = dtype == RSM_BF16 ? kRowVec<__hip_bfloat16> : kRowVec<float>, batch_vecs = 64 * kDeep;
  const size_t width = width_of(s, vocab);
  g.vecs = static_cast<unsigned>((width + vec - 1) / vec);
  g.batches_per_member = static_cast<int>((g.vecs + batch_vecs - 1) / batch_vecs);
  // Numbering the vectors through costs some instructions per vector; it pays where cutting every
  // member's part for itself would leave more than a seventh of the lanes idle.
  g.packed = static_cast<size_t>(g.batches_per_member) * batch_vecs * 7 > static_cast<size_t>(g.vecs) * 8;
  const int members = static_cast<int>((vocab + width - 1) / width) < s.team.size ? static_cast<int>((vocab + width - 1) / width) : s.team.size;
  const int64_t all = g.packed ? (static_cast<int64_t>(members) * g.vecs + batch_vecs - 1) / batch_vecs
                               : static_cast<int64_t>(members) * g.batches_per_member;
  g.batches = static_cast<int>(all);
  g.parts = 1;
  // Few rows: several workgroups to a row, so that the chip has some 1024 to run, four to a compute unit, but
  // each with eight batches, one for each of its waves, which then ranks them without reading them again.
  // Smaller shares lose more in the joining than they win, larger ones leave memory idle (512 workgroups of
  // four batches and more against 1024 of eight, 4 alternatives: 1 x 128000 bf16 over 8 members 10.7 and 10.3
  // us, 64 x 152000 15.4 and 13.7, 200 x 152000 25.2 and 23.1; 1 x 32000 9.3 and 9.7, 128 x 152000 18.8 and 19.6).
  if (rows && rows < 256) {
    int64_t parts = 1024 / static_cast<int64_t>(rows);
    const int64_t most = (all + kMaxWaves - 1) / kMaxWaves;
    if (parts > most) parts = most;
    if (parts > kMaxParts) parts = kMaxParts;
    g.parts = parts < 1 ? 1 : static_cast<int>(parts);
  }
  const int64_t mine = (all + g.parts - 1) / g.parts;
  // Many rows that are not long: half as many waves to a row and twice as many rows at a time, since a row's
  // waves stand idle while one of them ranks and joins (8 alternatives, 8 and 4 waves: 8192 x 20000 bf16 over 2
  // members 99.9 and 80.7 us, 8192 x 16000 74.0 and 68.3, 4096 x 50257 over 4 103 and 98; 4096 x 131072 over 8,
  // 64 batches, 186 and 187.  Without alternatives nobody ranks and the rule is worth little: 2048 x 32000 loses,
  // 27.2 and 28.7, 8192 x 20000 gains, 72.8 and 67.6.)
  const int most_waves = rows >= 2048 && all <= 32 ? kMaxWaves / 2 : kMaxWaves;
  g.waves = mine < most_waves ? static_cast<int>(mine) : most_waves;
  if (g.parts > 1) g.work_bytes = rows * g.parts * (sizeof(float4) + static_cast<size_t>(top_k) * 8);
  return g;
}

const char *moved(const void *p, int64_t bytes) { return p ? static_cast<const char *>(p) + bytes : nullptr; }
char *moved(void *p, int64_t bytes) { return p ? static_cast<char *>(p) + bytes : nullptr; }
template <typename T>
const T *moved_as(const void *p, int64_t bytes) {
  return reinterpret_cast<const T *>(moved(p, bytes));
}

template <typename T, bool kTop, bool kNt>
void launch_forward(const LogprobForward &p, bool packed, dim3 grid, int waves, hipStream_t st) {
  const dim3 block(static_cast<unsigned>(waves * 64));
  const size_t lds = shared_bytes(waves, kTop);
  const bool single = kTop && (p.batches + p.parts - 1) / p.parts <= waves;
  if (single && packed) hipLaunchKernelGGL((logprob_kernel<T, kTop, kNt, true, kTop>), grid, block, lds, st, p);
  else if (single) hipLaunchKernelGGL((logprob_kernel<T, kTop, kNt, false, kTop>), grid, block, lds, st, p);
  else if (packed) hipLaunchKernelGGL((logprob_kernel<T, kTop, kNt, true, false>), grid, block, lds, st, p);
  else hipLaunchKernelGGL((logprob_kernel<T, kTop, kNt, false, false>), grid, block, lds, st, p);
}

template <typename T>
void launch_forward(const LogprobForward &p, const LogprobPlan &g, dim3 grid, hipStream_t st, bool once) {
  if (p.top_k) {
    if (once) launch_forward<T, true, true>(p, g.packed, grid, g.waves, st);
    else launch_forward<T, true, false>(p, g.packed, grid, g.waves, st);
  } else {
    if (once) launch_forward<T, false, true>(p, g.packed, grid, g.waves, st);
    else launch_forward<T, false, false>(p, g.packed, grid, g.waves, st);
  }
}

template <typename T>
void launch_backward(const LogprobBackward &p, dim3 grid, hipStream_t st, bool large, bool packed) {
  const dim3 block(kGradLanes);
  if (packed) {
    if (large) hipLaunchKernelGGL((logprob_grad_kernel<T, true, true>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((logprob_grad_kernel<T, false, true>), grid, block, 0, st, p);
  } else {
    if (large) hipLaunchKernelGGL((logprob_grad_kernel<T, true, false>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((logprob_grad_kernel<T, false, false>), grid, block, 0, st, p);
  }
}

// 2^32 / n rounded up, 0 for 1.
unsigned per(unsigned n) { return n > 1 ? static_cast<unsigned>(((uint64_t{1} << 32) + n - 1) / n) : 0; }

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
  if (!a.logprob && !a.entropy && !a.lse && !a.largest && !a.log_sum && !a.top_ids && !a.top_logprobs) return rsm::fail("logprob_to_all: no result is asked for");
  if ((a.top_ids || a.top_logprobs) != (a.top_k > 0)) return rsm::fail("logprob_to_all: top_k and the arrays for the alternatives do not go together");
  if (!top_in_range(call, a.top_k, a.vocab) || !shape_of(a, call, &s)) return -1;
  const LogprobPlan g = plan_of(s, a.dtype, a.rows, a.vocab, a.top_k);
  if (g.parts > 1 && (!a.work || !a.pSync)) return rsm::fail("logprob_to_all: work (rsm_logprob_work_bytes) and pSync must be given for so few rows");
  if (a.rows == 0) return 0;
  const size_t size = type_size(a.dtype);
  rsm::Operands o(call);
  o.matrix(a.logits, "logits", a.rows, width_of(s, a.vocab), s.ld, size, false);
  o.add(a.tokens, "tokens", a.rows * 8, 8, false);
  o.add(a.logprob, "logprob", a.rows * 4, 4, true);
  o.add(a.entropy, "entropy", a.rows * 4, 4, true);
  o.add(a.lse, "lse", a.rows * 4, 4, true);
  o.add(a.largest, "largest", a.rows * 4, 4, true);
  o.add(a.log_sum, "log_sum", a.rows * 4, 4, true);
  o.add(a.top_ids, "top_ids", a.rows * a.top_k * 4, 4, true);
  o.add(a.top_logprobs, "top_logprobs", a.rows * a.top_k * 4, 4, true);
  if (g.parts > 1) {
    o.add(a.work, "work (rsm_logprob_work_bytes)", g.work_bytes, 16, true);
    o.add(a.pSync, "pSync (ROC_SHMEM_REDUCE_SYNC_SIZE longs)", ROC_SHMEM_REDUCE_SYNC_SIZE * sizeof(long), sizeof(long), true);
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
  p.largest = moved(a.largest, s.team.first);
  p.log_sum = moved(a.log_sum, s.team.first);
  p.top_ids = moved(a.top_ids, s.team.first);
  p.top_logprobs = moved(a.top_logprobs, s.team.first);
  p.batches = g.batches;
  p.batches_per_member = g.batches_per_member;
  p.vecs = g.vecs;
  p.per_vecs = per(g.vecs);
  p.parts = g.parts;
  if (g.parts > 1) {
    const size_t n = a.rows * g.parts;
    char *work = moved(a.work, s.team.first);
    p.part_sums = reinterpret_cast<float4 *>(work);
    p.part_keys = reinterpret_cast<uint64_t *>(work + n * sizeof(float4));
    p.arrived = reinterpret_cast<unsigned *>(moved(a.pSync, s.team.first));
  }
  const dim3 grid(static_cast<unsigned>(a.rows * g.parts));
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Logits that the Infinity Cache could not hold anyway are read past it: 4096 x 131072 bf16 without
  // alternatives 168 us against 186; smaller ones may still lie there from the product that made them.
  const bool once = a.rows * a.vocab * size > rsm::kInfinityCacheBytes;
  if (a.dtype == RSM_BF16) launch_forward<__hip_bfloat16>(p, g, grid, st, once);
  else launch_forward<float>(p, g, grid, st, once);
  return rsm::after_launch(call);
}

int rsm_logprob_to_all_grad(const rsm_logprob_grad_args_t *args, void *stream) {
  RSM_ENTRY;
  const char *call = "logprob_to_all_grad";
  if (!args) return rsm::fail("logprob_to_all_grad: arguments are NULL");
  const rsm_logprob_grad_args_t &a = *args;
  LogprobShape s;
  if (!a.largest != !a.log_sum) return rsm::fail("logprob_to_all_grad: largest and log_sum go together");
  if (!a.logits || !a.grad_logits || !(a.lse || a.log_sum))
    return rsm::fail("logprob_to_all_grad: logits, grad_logits and lse (or largest and log_sum) must be given");
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
  const int logits = o.matrix(a.logits, "logits", a.rows, width, s.ld, size, false);
  o.add(a.tokens, "tokens", a.rows * 8, 8, false);
  o.add(a.lse, "lse", a.rows * 4, 4, false);
  o.add(a.largest, "largest", a.rows * 4, 4, false);
  o.add(a.log_sum, "log_sum", a.rows * 4, 4, false);
  o.add(a.entropy, "entropy", a.rows * 4, 4, false);
  o.add(a.grad_logprob, "grad_logprob", a.rows * 4, 4, false);
  o.add(a.grad_entropy, "grad_entropy", a.rows * 4, 4, false);
  o.add(a.grad_lse, "grad_lse", a.rows * 4, 4, false);
  o.matrix(a.grad_logits, "grad_logits", a.rows, width, grad_ld, size, true, grad_ld == s.ld ? logits : o.kNone);
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
  p.largest = moved_as<float>(a.largest, s.team.first);
  p.normaliser = moved_as<float>(a.log_sum ? a.log_sum : a.lse, s.team.first);
  p.entropy = moved_as<float>(a.entropy, s.team.first);
  p.grad_logprob = moved_as<float>(a.grad_logprob, s.team.first);
  p.grad_entropy = moved_as<float>(a.grad_entropy, s.team.first);
  p.grad_lse = moved_as<float>(a.grad_lse, s.team.first);
  p.grad_logits = moved(a.grad_logits, s.team.first);
  const size_t vec = a.dtype == RSM_BF16 ? kRowVec<__hip_bfloat16> : kRowVec<float>, most = kGradLanes * kGradDeep;
  p.vecs = static_cast<unsigned>((width + vec - 1) / vec);
  p.chunks = static_cast<int>((p.vecs + most - 1) / most);
  p.per_vecs = per(p.vecs);
  p.per_members = per(static_cast<unsigned>(p.members));
  // Short lines would leave a workgroup without enough to do for its start: 4096 x 1000 bf16 over 8 members
  // 173 us by lines and 16 numbered through.  Longer ones pay more for numbering (a row's numbers are
  // read for every vector) than for lanes that have nothing to do.
  const bool packed = p.vecs < 512;
  const size_t lines = a.rows * p.members;
  const size_t wgs = packed ? (lines * p.vecs + most - 1) / most : lines * static_cast<size_t>(p.chunks);
  const size_t x = wgs < 0x800000 ? wgs : 0x800000, y = (wgs + x - 1) / x;
  if (y > 65535) return rsm::fail("logprob_to_all_grad: too many rows for one launch");
  const dim3 grid(static_cast<unsigned>(x), static_cast<unsigned>(y));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool large = 2 * a.rows * a.vocab * size > rsm::kInfinityCacheBytes;
  if (a.dtype == RSM_BF16) launch_backward<__hip_bfloat16>(p, grid, st, large, packed);
  else launch_backward<float>(p, grid, st, large, packed);
  return rsm::after_launch(call);
}

}  // extern "C"
