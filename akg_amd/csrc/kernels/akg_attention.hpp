/**
 * Attention for gfx950 that keeps no probabilities: the forward pass with the running maximum and sum of a softmax, and
 * the backward pass, which recomputes the probabilities from the log of that sum.
 *
 *   s = scale q k^T (+ mask), lse = log sum_j exp s, out = exp(s - lse) v
 *   delta = rowsum(dout out), p = exp(s - lse), ds = p (dout v^T - delta)
 *   dv = p^T dout, dq = scale ds k, dk = scale ds^T q
 *
 * Every product runs on v_mfma_f32_32x32x16 with float32 accumulators. A wavefront owns 32 rows (queries, or keys in the
 * kernel of dk and dv) as the COLUMNS of its MFMA results: lane n and n + 32 hold row n, so that the maximum, the sum and
 * the rescaling of a row are values of one lane pair, and the probabilities that one MFMA leaves in a lane are already the
 * operand of the next one. A lane holds of every 16 contracted positions those 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3
 * (h = lane / 32); the order of contracted positions does not matter as long as both operands have the same, and the
 * transposing LDS reads fetch four adjacent positions each, so nothing is exchanged between lanes.
 *
 * The other side's tiles lie in LDS as they lie in memory (rows of channels). They are read two ways: along the row
 * (16 bytes of a row per lane) and transposed (ds_read_b64_tr_b16: four rows of 16 columns per sixteen lanes). Rows are an
 * odd multiple of 64 bytes apart, so four neighbouring rows of 64 bytes cover the 256 bytes of the banks (transposed
 * reads), and the 16-byte chunks inside 64 bytes are permuted by (row / 4) % 4, so the sixteen rows that a 128-bit read
 * serves at a time (the lane quads 0, 3, 5, 6 of a half wavefront, then 1, 2, 4, 7) fall into different bank groups. (Rows
 * without padding and whole units permuted by the row are as free of conflicts, but every read then has an address of its
 * own instead of an offset: eight to sixteen registers more, which the kernels of 128 channels spill.)
 *
 * Heads that share keys are rows of one problem: row r of a key head is query r / G of head r % G, so the tiles of keys
 * and values are fetched once for the group, and the gradients of keys and values are sums without atomics.
 */
#pragma once

namespace akg {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef u32 u32x4 __attribute__((ext_vector_type(4)));
typedef u32 u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct BF16 {
  typedef bf16 dtype;
  static constexpr bool kNarrowRange = false;
  typedef __bf16 frag __attribute__((ext_vector_type(8)));
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  static AKG_DEV f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
  static AKG_DEV u32 pack(float lo, float hi) {
    const pair p = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
    return __builtin_bit_cast(u32, p);
  }
  static AKG_DEV float low(u32 w) { return __builtin_bit_cast(float, w << 16); }
  static AKG_DEV float high(u32 w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
};
struct F16 {
  typedef f16 dtype;
  static constexpr bool kNarrowRange = true;
  typedef _Float16 frag __attribute__((ext_vector_type(8)));
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  static AKG_DEV f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
  }
  static AKG_DEV u32 pack(float lo, float hi) {
    const pair p = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(u32, p);
  }
  static AKG_DEV float low(u32 w) { return static_cast<float>(__builtin_bit_cast(pair, w)[0]); }
  static AKG_DEV float high(u32 w) { return static_cast<float>(__builtin_bit_cast(pair, w)[1]); }
};

template <int N>
struct IntTag {
  static constexpr int value = N;
};
// f(0) ... f(N - 1) with constants: what a loop that the compiler may decide not to unroll cannot promise.
template <int N, int I = 0, typename F>
AKG_DEV void unrolled(F &&f) {
  if constexpr (I < N) {
    f(IntTag<I>());
    unrolled<N, I + 1>(f);
  }
}

constexpr float kLog2e = 0x1.715476p+0f, kLn2 = 0x1.62e430p-1f;
constexpr int kRows = 32;      // rows of a wavefront
constexpr int kTile = 64;      // keys of a tile (forward, dq)
constexpr int kTileRows = 32;  // queries of a tile (dk, dv)

constexpr int padded(int d) { return (d + 31) / 32 * 32; }
constexpr int pitch(int d) { return padded(d) / 32 % 2 == 1 ? padded(d) * 2 : padded(d) * 2 + 64; }
// Byte of chunk `chunk` (16 bytes) of row `row` in a tile of D channels.
template <int D>
AKG_DEV int chunk_at(int row, int chunk) {
  return row * pitch(D) + ((chunk ^ ((row >> 2) & 3)) << 4);
}
// Keys that are only read along the row: rows an odd number of chunks apart.
constexpr int own_pitch(int d) { return padded(d) * 2 + 16; }

AKG_DEV float neg_inf() { return -__builtin_inff(); }
// The two halves of a row's lane pair (n and n + 32) joined.
AKG_DEV float max_halves(float v) {
  const u32 w = __builtin_bit_cast(u32, v);
  const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __builtin_fmaxf(__builtin_bit_cast(float, static_cast<u32>(s[0])), __builtin_bit_cast(float, static_cast<u32>(s[1])));
}
AKG_DEV float add_halves(float v) {
  const u32 w = __builtin_bit_cast(u32, v);
  const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __builtin_bit_cast(float, static_cast<u32>(s[0])) + __builtin_bit_cast(float, static_cast<u32>(s[1]));
}

// ---- what the emitted kernel states about its description -------------------------------------------------------------
// Extents that are kernel arguments, and what follows from them.
struct Extents {
  long batch, sq, sk;
};

// MASK: 0 none, 1 bool (true: the pair counts), 2 float16, 3 bfloat16, 4 float32 (added to the scaled score).
template <typename T_, int DK_, int DV_, int HKV_, int G_, bool HEADS_FIRST_, bool CAUSAL_, int MASK_, bool MASK_B_, bool MASK_H_, bool MASK_Q_>
struct Config {
  typedef T_ T;
  static constexpr int DK = DK_, DV = DV_, HKV = HKV_, G = G_, H = HKV_ * G_, MASK = MASK_;
  static constexpr bool HEADS_FIRST = HEADS_FIRST_, CAUSAL = CAUSAL_;
  // which leading dimensions of the mask are the scores' (the others have extent 1)
  static constexpr bool MASK_B = MASK_B_, MASK_H = MASK_H_, MASK_Q = MASK_Q_;
  // Scores are exponents of 2 (scale log2 e in one factor), unless a mask is added: its lowest values times log2 e would
  // leave float32, so sums of score and mask, and their maxima, are kept as they are and differences are multiplied.
  static constexpr bool ADDED = MASK_ >= 2;
};

// Where the rows of one key head lie, in bytes: row r = query r / G of head r % G.
template <typename C, int D>
struct RowsOf {
  const char *base;     // of (batch, first head of the group)
  long stepI, stepG;    // from query to query, from head to head
  AKG_DEV RowsOf(const void *p, long b, long hkv, const Extents &e) {
    if (C::HEADS_FIRST) {
      stepI = 2L * D;
      stepG = 2L * D * e.sq;
      base = static_cast<const char *>(p) + (b * C::H + hkv * C::G) * stepG;
    } else {
      stepI = 2L * D * C::H;
      stepG = 2L * D;
      base = static_cast<const char *>(p) + (b * e.sq) * stepI + hkv * C::G * stepG;
    }
  }
  AKG_DEV long offset(long r) const { return r / C::G * stepI + r % C::G * stepG; }
};
template <typename C, int D>
struct KeysOf {
  const char *base;
  long step;
  AKG_DEV KeysOf(const void *p, long b, long hkv, const Extents &e) {
    step = C::HEADS_FIRST ? 2L * D : 2L * D * C::HKV;
    base = static_cast<const char *>(p) + (C::HEADS_FIRST ? (b * C::HKV + hkv) * e.sk * step : b * e.sk * step + hkv * 2L * D);
  }
};

// How many keys query i sees, given the lengths of its sequence (none behind the queries' length).
template <typename C>
AKG_DEV int keys_seen(long i, int ql, int kl) {
  if (i >= ql) return 0;
  if (!C::CAUSAL) return kl;
  const int n = static_cast<int>(i) + kl - ql + 1;
  return n < 0 ? 0 : (n < kl ? n : kl);
}

template <typename C>
AKG_DEV int clamped_length(const int *lengths, long b, long most) {
  if (lengths == nullptr) return static_cast<int>(most);
  const long n = lengths[b];
  return static_cast<int>(n < 0 ? 0 : (n < most ? n : most));
}

// ---- tiles in LDS -----------------------------------------------------------------------------------------------------
// A tile of ROWS rows of D 16-bit channels on its way from memory to LDS through the registers of THREADS threads.
template <int ROWS, int D, int THREADS>
struct TileLoad {
  static constexpr int kPerRow = D / 8;
  static constexpr int kChunks = ROWS * kPerRow;
  static constexpr int kEach = (kChunks + THREADS - 1) / THREADS;
  static constexpr bool kWhole = kChunks % THREADS == 0;
  u32x4 held[kEach];
  // `offset(row)`: byte offset of the row from the descriptor's base, or kBeyondEveryBuffer (reads zeros).
  template <typename F>
  AKG_DEV void load(Buffer buf, int tid, F offset) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int c = tid + i * THREADS;
      const u32 off = offset(c / kPerRow) + static_cast<u32>(c % kPerRow) * 16u;
      held[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(buf, (kWhole || c < kChunks) ? off : kBeyondEveryBuffer, 0, 0));
    }
  }
  template <bool OWN = false>
  AKG_DEV void store(u8 *tile, int tid) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int c = tid + i * THREADS;
      const int row = c / kPerRow, chunk = c % kPerRow;
      if (kWhole || c < kChunks) *reinterpret_cast<u32x4 *>(tile + (OWN ? row * own_pitch(D) + chunk * 16 : chunk_at<D>(row, chunk))) = held[i];
    }
  }
};

// A lane's places in a tile of D channels. What differs between the reads of a tile is then a constant offset (left to
// itself the compiler keeps an address per read).
template <int D>
struct Reader {
  int along[2], across[2];
  AKG_DEV explicit Reader(int lane) {
    const int row = lane & 31, h = lane >> 5;
    along[0] = chunk_at<D>(row, h);
    along[1] = chunk_at<D>(row, 2 + h);
    const int i = lane & 15, r = 4 * h + (i >> 2), chunk = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    across[0] = chunk_at<D>(r, chunk) + (i & 1) * 8;
    across[1] = chunk_at<D>(r + 8, chunk) + (i & 1) * 8;
  }
  // 16 bytes of row `row0 + lane % 32` (row0 a multiple of 32): channels 16 c + 8 (lane / 32) ... + 7, the operand of 16
  // contracted channels.
  AKG_DEV u32x4 row(const u8 *tile, int row0, int c) const {
    return *reinterpret_cast<const u32x4 *>(tile + along[c & 1] + (row0 * pitch(D) + 64 * (c >> 1)));
  }
  // Column 32 dt + lane % 32 of the rows row0 + 4 h .. 4 h + 3 and row0 + 8 + 4 h .. (h = lane / 32; row0 a multiple of 16).
  AKG_DEV u32x4 transposed(const u8 *tile, int row0, int dt) const {
    const int more = row0 * pitch(D) + 64 * dt;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(tile + across[0] + more));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(tile + across[1] + more));
    const u32x2 l = __builtin_bit_cast(u32x2, lo), u = __builtin_bit_cast(u32x2, hi);
    return u32x4{l[0], l[1], u[0], u[1]};
  }
};
template <int D>
AKG_DEV u32x4 read_own(const u8 *keys, int row0, int c, int lane) {
  return *reinterpret_cast<const u32x4 *>(keys + (row0 + (lane & 31)) * own_pitch(D) + ((lane >> 5) << 4) + 32 * c);
}
// The channels behind D of a tile's rows (D to the next multiple of 32) hold zeros: written once, never again.
template <int ROWS, int D, int THREADS>
AKG_DEV void clear_padding(u8 *tile, int tid) {
  if constexpr (D % 32 != 0) {
    constexpr int kPad = (padded(D) - D) / 8;
    for (int c = tid; c < ROWS * kPad; c += THREADS) {
      const int row = c / kPad, chunk = D / 8 + c % kPad;
      *reinterpret_cast<u32x4 *>(tile + chunk_at<D>(row, chunk)) = u32x4{0, 0, 0, 0};
    }
  }
}

// The operand of a wavefront's own 32 rows, straight from memory (channels behind D: zeros).
template <int D>
AKG_DEV void load_own(const char *row, bool ok, int lane, u32x4 (&own)[(D + 15) / 16]) {
#pragma unroll
  for (int c = 0; c < (D + 15) / 16; ++c) {
    const int at = 16 * c + 8 * (lane >> 5);
    own[c] = (ok && (D % 16 == 0 || at < D)) ? *reinterpret_cast<const u32x4 *>(row + 2 * at) : u32x4{0, 0, 0, 0};
  }
}

AKG_DEV u32 records(long bytes) { return static_cast<u32>(bytes < 0 ? 0 : (bytes < 0x7fffffffL ? bytes : 0x7fffffffL)); }

template <bool B, typename X, typename Y>
struct conditional {
  typedef X type;
};
template <typename X, typename Y>
struct conditional<false, X, Y> {
  typedef Y type;
};

// ---- masks ------------------------------------------------------------------------------------------------------------
template <typename C>
AKG_DEV long mask_row(long b, long h, long i, const Extents &e) {
  long r = 0;
  if (C::MASK_B) r = b;
  if (C::MASK_H) r = r * C::H + h;
  if (C::MASK_Q) r = r * e.sq + i;
  return r * e.sk;
}
// The score with the mask at element `at` applied; `factor`: scale log2 e, or the scale where the mask is added.
template <typename C>
AKG_DEV float with_mask(float s, float factor, const void *mask, long at) {
  if constexpr (C::MASK == 1) return static_cast<const u8 *>(mask)[at] ? s * factor : neg_inf();
  if constexpr (C::MASK == 2) return __builtin_fmaf(s, factor, f16::load(static_cast<const f16::storage *>(mask)[at]));
  if constexpr (C::MASK == 3) return __builtin_fmaf(s, factor, bf16::load(static_cast<const bf16::storage *>(mask)[at]));
  if constexpr (C::MASK == 4) return __builtin_fmaf(s, factor, static_cast<const float *>(mask)[at]);
  return s * factor;
}
// The mask's row of one query, 32 keys at a time: a lane holds four groups of four adjacent ones (as of the scores), requested
// before the scores are computed, in wide loads that run on into the next row (no score takes what they find there). Where
// they would pass the end of the mask they are moved back instead, and `fix` loads one element at a time: in a branch that
// waits for itself, where the scores are. (With loads in two branches the compiler waited for those of the keys ahead at
// every use: 4 x 1000 x 1003 x 16 x 64, inputs in the last cache, took 54 us instead of 49 when that was tried.)
__device__ const u32 kNothing[32] = {};
template <typename C>
struct MaskRow {
  typedef conditional<C::MASK == 1, u8, typename conditional<C::MASK == 4, float, u16>::type> Choice;
  typedef typename Choice::type E;
  typedef E E4 __attribute__((ext_vector_type(4)));
  typedef E4 Unaligned __attribute__((aligned(sizeof(E))));
  typedef __attribute__((address_space(1))) const Unaligned Global;   // (either pointer's memory)
  const E *row, *wide;
  int keys, room;   // of the row, and to the end of the mask
  struct Part {
    E4 value[4];
    AKG_DEV float apply(float s, float factor, int r) const {
      const E one = value[r >> 2][r & 3];
      return with_mask<C>(s, factor, &one, 0);
    }
  };
  AKG_DEV MaskRow(const void *mask, long at, const Extents &e) : row(static_cast<const E *>(mask) + at), keys(static_cast<int>(e.sk)) {
    const long all = (C::MASK_B ? e.batch : 1) * (C::MASK_H ? C::H : 1) * (C::MASK_Q ? e.sq : 1) * e.sk - at;
    room = all < 0x40000000 ? static_cast<int>(all) : 0x40000000;
    wide = room < 32 ? reinterpret_cast<const E *>(kNothing) : row;
  }
  AKG_DEV Part part(int j0, int half) const {
    const int within = j0 < room - 32 ? j0 : room - 32;
    const E *from = wide + (within > 0 ? within : 0) + 4 * half;
    Part p;
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) p.value[r4] = *(Global *)(from + 8 * r4);
    return p;
  }
  AKG_DEV void fix(Part &p, int j0, int half) const {
    if (!__any(j0 + 32 > room)) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = j0 + 8 * (r >> 2) + 4 * half + (r & 3);
      p.value[r >> 2][r & 3] = row[j < keys ? j : keys - 1];
    }
    u32 words[sizeof(Part) / 4];   // (waited for here)
    __builtin_memcpy(words, &p, sizeof(Part));
#pragma unroll
    for (unsigned w = 0; w < sizeof(Part) / 4; ++w) asm volatile("" : "+v"(words[w]));
    __builtin_memcpy(&p, words, sizeof(Part));
  }
};
// 2^x or e^x of a difference of scores, and a row's log of the sum from its maximum and its sum.
template <typename C>
AKG_DEV float power(float x) {
  return __builtin_amdgcn_exp2f(C::ADDED ? x * kLog2e : x);
}
template <typename C>
AKG_DEV float log_sum(float top, float sum) {
  const float l = __builtin_amdgcn_logf(sum);
  return sum == 0.0f ? neg_inf() : C::ADDED ? __builtin_fmaf(l, kLn2, top) : (top + l) * kLn2;
}

// ---- workgroup -> (key head, tile) ------------------------------------------------------------------------------------
// Workgroups go round robin to the 8 XCDs. With a multiple of 8 key heads (over the batch) a head stays on one XCD, whose
// L2 then holds its keys and values once; else heads follow one another. Tiles in the given order, heads inside.
AKG_DEV void head_and_tile(long id, long heads, long &head, long &tile) {
  if (heads % 8 == 0) {
    const long each = heads / 8, y = id / 8;
    head = id % 8 + 8 * (y % each);
    tile = y / each;
  } else {
    head = id % heads;
    tile = id / heads;
  }
}

// Order of a block of MF matrix instructions fed by RD LDS reads: LEAD reads ahead, then after every matrix instruction its
// share of the others. (Left to itself the compiler issues a read right in front of its use, and the matrix cores wait.)
template <int MF, int RD, int LEAD, int M = 0>
struct FeedOrder {
  static constexpr int kLead = LEAD < RD ? LEAD : RD;
  static constexpr int kEach = (RD - kLead + MF - 1) / (MF > 0 ? MF : 1);
  static constexpr int kFrom = M * kEach < RD - kLead ? M * kEach : RD - kLead;
  static constexpr int kUpto = (M + 1) * kEach < RD - kLead ? (M + 1) * kEach : RD - kLead;
  static AKG_DEV void emit() {
    if constexpr (M == 0) __builtin_amdgcn_sched_group_barrier(0x100, kLead, 0);
    if constexpr (M < MF) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if constexpr (kUpto > kFrom) __builtin_amdgcn_sched_group_barrier(0x100, kUpto - kFrom, 0);
      FeedOrder<MF, RD, LEAD, M + 1>::emit();
    }
  }
};

// ---- ranges of keys that several workgroups share -----------------------------------------------------------------------
// Every range leaves accumulators, maximum and sum of its rows in the workspace; the workgroup that arrives last at the
// counter of its rows joins them, in the order of the ranges whoever that is (a second launch costs 3 to 6 us more).
// Workspace: the counters, to the next 256 bytes; accumulators [ranges][rows of all key heads][padded channels]; then
// (maximum, sum) [ranges][rows].
template <typename C>
struct Ranges {
  Buffer ws;
  unsigned *counters;
  long rows;      // of all key heads
  int splits;
  u32 accumulators, states;
  AKG_DEV Ranges(float *workspace, long groups, long all, int n) : counters(reinterpret_cast<unsigned *>(workspace)), rows(all), splits(n) {
    accumulators = static_cast<u32>((groups * 4 + 255) / 256 * 256);
    states = accumulators + static_cast<u32>(n * all * padded(C::DV) * 4);
    ws = make_buffer(workspace, states + n * all * 8L);   // (below 2 GiB: checked by the host)
  }
  AKG_DEV u32 accumulator(long s, long row, int d) const { return accumulators + static_cast<u32>(((s * rows + row) * padded(C::DV) + d) * 4); }
  AKG_DEV u32 state(long s, long row) const { return states + static_cast<u32>((s * rows + row) * 8); }
};

// Rows row0 .. row0 + count - 1 (of one key head, `at` that of row0 among all) from their ranges. Of a row, a thread takes four
// channels of every `sharers`-th range, four ranges requested at a time; sharers meet in LDS that the workgroup needs no more.
template <int THREADS>
struct Meeting {
  f32x4 parts[THREADS];
  float tops[THREADS], sums[THREADS];
  unsigned flag;   // of last_workgroup
};
template <typename C, int THREADS>
AKG_DEV void join(const Ranges<C> &in, Meeting<THREADS> &meet, long b, long hkv, long row0, long at, int count, void *out, float *lse,
                  const Extents &e, int tid) {
  typedef typename C::T T;
  constexpr int DV = C::DV, kPer = DV / 4, kAtOnce = 4;
  int sharers = 1;
  while (sharers < 8 && 2 * sharers * kPer * count <= THREADS && 2 * sharers <= in.splits) sharers *= 2;
  const int per = kPer * sharers, together = THREADS / per, first = tid % per / kPer, d = tid % kPer * 4;
  const RowsOf<C, DV> orows(out, b, hkv, e);
  for (int r0 = 0; r0 < count; r0 += together) {
    const int r = r0 + tid / per;
    const bool mine = tid < together * per && r < count;
    float top = neg_inf(), sum = 0.0f;
    f32x4 acc = {};
    for (int s0 = first; mine && s0 < in.splits; s0 += sharers * kAtOnce) {
      float x[kAtOnce][4], t[kAtOnce][2];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {   // (behind the last range: zeros)
        const int s = s0 + u * sharers;
        ws_load_chunk_if<2>(in.ws, s < in.splits, in.state(s, at + r), t[u]);
        ws_load_chunk_if<4>(in.ws, s < in.splits, in.accumulator(s, at + r, d), x[u]);
      }
      float m = top;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (t[u][1] == 0.0f) {   // (a range without keys wrote no accumulators)
          t[u][0] = neg_inf();
#pragma unroll
          for (int z = 0; z < 4; ++z) x[u][z] = 0.0f;
        }
        m = __builtin_fmaxf(m, t[u][0]);
      }
      const float base = m == neg_inf() ? 0.0f : m, old = power<C>(top - base);
      top = m;
      sum *= old;
      acc *= old;
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const float w = power<C>(t[u][0] - base);
        sum = __builtin_fmaf(t[u][1], w, sum);
#pragma unroll
        for (int z = 0; z < 4; ++z) acc[z] = __builtin_fmaf(x[u][z], w, acc[z]);
      }
    }
    if (sharers > 1) {
      if (r0 > 0) __syncthreads();
      meet.parts[tid] = acc;
      meet.tops[tid] = top;
      meet.sums[tid] = sum;
      __syncthreads();
      if (mine && first == 0) {
        for (int g = 1; g < sharers; ++g) top = __builtin_fmaxf(top, meet.tops[tid + g * kPer]);
        const float base = top == neg_inf() ? 0.0f : top;
        sum = 0.0f;
        acc = f32x4{};
        for (int g = 0; g < sharers; ++g) {
          const float w = power<C>(meet.tops[tid + g * kPer] - base);
          sum = __builtin_fmaf(meet.sums[tid + g * kPer], w, sum);
          const f32x4 x = meet.parts[tid + g * kPer];
#pragma unroll
          for (int z = 0; z < 4; ++z) acc[z] = __builtin_fmaf(x[z], w, acc[z]);
        }
      }
    }
    if (!mine || first != 0) continue;
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const long row = row0 + r;
    u32x2 w;
    w[0] = T::pack(acc[0] * inverse, acc[1] * inverse);
    w[1] = T::pack(acc[2] * inverse, acc[3] * inverse);
    *reinterpret_cast<u32x2 *>(const_cast<char *>(orows.base) + orows.offset(row) + 2 * d) = w;
    if (lse != nullptr && d == 0) lse[(b * C::H + hkv * C::G + row % C::G) * e.sq + row / C::G] = log_sum<C>(top, sum);
  }
}

// A launch of its own that joins, ROWS rows of a key head a workgroup; the ranges' workgroups had GROUP rows each.
template <typename C, int ROWS, int GROUP>
AKG_DEV void join_rows(float *ws, void *out, float *lse, const Extents &e, int splits) {
  __shared__ Meeting<256> meet;
  const long rows = e.sq * C::G, tiles = (rows + ROWS - 1) / ROWS, head = blockIdx.x / tiles, row0 = blockIdx.x % tiles * ROWS;
  const Ranges<C> ranges(ws, e.batch * C::HKV * ((rows + GROUP - 1) / GROUP), e.batch * C::HKV * rows, splits);
  join<C, 256>(ranges, meet, head / C::HKV, head % C::HKV, row0, head * rows + row0, static_cast<int>(rows - row0 < ROWS ? rows - row0 : ROWS), out, lse, e, static_cast<int>(threadIdx.x));
}

// ---- forward ----------------------------------------------------------------------------------------------------------
// SPLIT: the workgroup takes one of `splits` ranges of the keys (Ranges). JOIN: the last one joins them.
//
// Many rows are bound by the matrix units and by the issue of what stands beside them: 2 x 4096 queries and keys, 32 heads over
// 8 of 128 channels, causal, bfloat16, take 301 us, 0.91 PFLOP/s (a matrix product of 8192 each way reaches 1.36); the
// matrix instructions alone would take 215, the vector instructions alone 151. Few rows are bound by the keys and values from
// memory: one query of 8 sequences over 8192 keys takes 51 us, 4.0 TB/s, and 44 where the last level cache still holds part
// of them. Tried for both and left out: a second set of tiles under way (token 54, training unchanged), 64 rows a wavefront,
// four wavefronts a workgroup and two workgroups a CU (training 382), raised wave priority around the matrix instructions.
template <typename C, int NW, bool SPLIT, bool JOIN>
AKG_DEV void forward(const void *q, const void *k, const void *v, const void *mask, const int *qlens, const int *klens,
                     void *out, float *lse, float *ws, Extents e, float scale, int splits) {
  typedef typename C::T T;
  constexpr int DK = C::DK, DV = C::DV, CK = (DK + 15) / 16, TV = padded(DV) / 32, kThreads = 64 * NW, kGroup = kRows * NW;
  // A third tile, where a CU holds one workgroup anyway, spares a barrier: what is being written no wavefront reads.
  constexpr int kTiles = NW == 8 && 3 * kTile * (pitch(DK) + pitch(DV)) <= 160 * 1024 ? 3 : 2;
  struct Lds {
    u8 ktiles[kTiles][kTile * pitch(DK)], vtiles[kTiles][kTile * pitch(DV)];
  };
  __shared__ __attribute__((aligned(16))) Lds lds;
  static_assert(sizeof(Lds) >= sizeof(Meeting<kThreads>), "the join meets where the tiles were");
  auto &ktiles = lds.ktiles;
  auto &vtiles = lds.vtiles;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const long rows = e.sq * C::G, tiles = (rows + kGroup - 1) / kGroup, heads = e.batch * C::HKV;
  long id = blockIdx.x;
  const int split = SPLIT ? static_cast<int>(id % splits) : 0;
  if (SPLIT) id /= splits;
  long head, tile;
  head_and_tile(id, heads, head, tile);
  tile = tiles - 1 - tile;   // the rows that see most keys first
  const long b = head / C::HKV, hkv = head % C::HKV;
  const int ql = clamped_length<C>(qlens, b, e.sq), kl = clamped_length<C>(klens, b, e.sk);

  const long row0 = tile * kGroup;
  // keys of the workgroup: those of its last row that has any
  long last = (row0 + kGroup < rows ? row0 + kGroup : rows) - 1;
  long lastI = last / C::G;
  if (lastI >= ql) lastI = ql - 1;
  const int most = row0 / C::G < ql ? keys_seen<C>(lastI, ql, kl) : 0;
  int first = 0, end = most;
  if (SPLIT) {
    const int all = (most + kTile - 1) / kTile, each = (all + splits - 1) / splits;
    first = split * each * kTile < most ? split * each * kTile : most;   // (most + 64 kTile stays below 2^31: checked by the host)
    end = first + each * kTile < most ? first + each * kTile : most;
  }

  const RowsOf<C, DK> qrows(q, b, hkv, e);
  const float c = C::ADDED ? scale : scale * kLog2e;
  const long row = row0 + wave * kRows + (lane & 31), i = row / C::G;
  const bool exists = row < rows;
  const int seen = exists ? keys_seen<C>(i, ql, kl) : 0;
  u32x4 own[CK];
  load_own<DK>(qrows.base + qrows.offset(exists ? row : 0), seen > 0, lane, own);
  f32x16 acc[TV];
#pragma unroll
  for (int d = 0; d < TV; ++d) acc[d] = {};
  float top = neg_inf(), sum[2] = {0.0f, 0.0f};   // the row's maximum (or a little less); sums over this lane's keys
  const MaskRow<C> maskRow(mask, C::MASK != 0 ? mask_row<C>(b, hkv * C::G + row % C::G, exists ? i : 0, e) : 0, e);

  const KeysOf<C, DK> keys(k, b, hkv, e);
  const KeysOf<C, DV> values(v, b, hkv, e);
  const Reader<DK> kread(lane);
  const Reader<DV> vread(lane);
  TileLoad<kTile, DK, kThreads> kload;
  TileLoad<kTile, DV, kThreads> vload;
  auto fetch = [&](int k0) {
    // (rows behind the keys' length lie behind the descriptor and read zeros)
    const Buffer kb = make_buffer(keys.base + k0 * keys.step, records((kl - k0 - 1) * keys.step + 2 * DK));
    const Buffer vb = make_buffer(values.base + k0 * values.step, records((kl - k0 - 1) * values.step + 2 * DV));
    kload.load(kb, tid, [&](int r) { return static_cast<u32>(r * static_cast<int>(keys.step)); });
    vload.load(vb, tid, [&](int r) { return static_cast<u32>(r * static_cast<int>(values.step)); });
  };
#pragma unroll
  for (int x = 0; x < kTiles; ++x) {
    clear_padding<kTile, DK, kThreads>(ktiles[x], tid);
    clear_padding<kTile, DV, kThreads>(vtiles[x], tid);
  }
  if (first < end) {   // (two tiles, both asked for before the first is waited for)
    fetch(first);
    const TileLoad<kTile, DK, kThreads> know = kload;
    const TileLoad<kTile, DV, kThreads> vnow = vload;
    fetch(first + kTile < end ? first + kTile : kl);
    know.store(ktiles[0], tid);
    vnow.store(vtiles[0], tid);
    kload.store(ktiles[1], tid);
    vload.store(vtiles[1], tid);
  }
  __syncthreads();

  f32x16 s;                 // scores of 32 keys
  float peak = neg_inf();   // the largest of them (of this lane's keys)
  typename MaskRow<C>::Part part, later;   // what the mask says of these 32 keys and the next (requested 64 keys ahead)
  // What the mask, the lengths and the causal order leave of the scores of the keys from j0 on, and their largest.
  auto limit = [&](int j0, f32x16 &x) {
    float m = neg_inf();
    if (C::MASK != 0) maskRow.fix(part, j0, half);
#pragma unroll
    for (int r = 0; C::MASK != 0 && r < 16; ++r) x[r] = part.apply(x[r], c, r);
    if (__any(j0 + 32 > seen)) {
      const int left = seen - j0 - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[r] = 8 * (r >> 2) + (r & 3) < left ? x[r] : neg_inf();
        asm volatile("" : "+v"(x[r]));   // (a branch: the compiler would compare and select for every tile)
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) m = __builtin_fmaxf(m, x[r]);
    return m;
  };
  // The keys from j0 on, whose scores are in `s`: their probabilities, while the scores of the 32 keys behind them are
  // computed (rows `krow` of `kt`; of whatever lies there where no row sees more), and their part of the result. One stream
  // without branches around it: with the two cases apart the accumulators were held twice.
  auto step = [&](int j0, const u8 *vt, int vrow, const u8 *kt, int krow) {
    // The maximum that the exponents are taken against follows the scores only when they are 2^8 above it: sums and
    // accumulators then have to be rescaled, which most tiles are spared; what is kept is as exact against any maximum.
    // float16 takes probabilities up to 2^15 (2^7 at the maximum found, 2^8 above that): the weights of a long tail, each a
    // small part of the largest, then have their digits down to 2^-21 of it.
    constexpr float kUnder = !T::kNarrowRange ? 0.0f : C::ADDED ? 7.0f * kLn2 : 7.0f;
    float m = max_halves(peak);
    m = C::MASK == 0 ? __builtin_fmaf(m, c, -kUnder) : m - kUnder;
    if (__any(m > top + (C::ADDED ? 5.5f : 8.0f))) {
      m = __builtin_fmaxf(top, m);
      const float shrink = power<C>(top - (m == neg_inf() ? 0.0f : m));
      top = m;
      sum[0] *= shrink;
      sum[1] *= shrink;
#pragma unroll
      for (int d = 0; d < TV; ++d) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] *= shrink;
      }
    }
    const float base = top == neg_inf() ? 0.0f : top;
    if (C::MASK != 0) {
      part = later;
      later = maskRow.part(j0 + 64, half);
    }
    // Probabilities are rounded to the type of the values for the matrix units (half a step of at most 2^-9 each, of
    // changing sign; the sum has them unrounded). A matrix instruction keeps its unit busy for 32 cycles and the issue for
    // four: a few vector instructions behind each of them, and operands read four ahead. (The barriers keep that order.)
    constexpr int kLead = 4, kEach = (16 + CK - 1) / CK;
    u32x4 p[2], a[CK];
    f32x16 next = {};
#pragma unroll
    for (int x = 0; x < kLead && x < CK; ++x) a[x] = kread.row(kt, krow, x);
#pragma unroll
    for (int x = 0; x < CK; ++x) {
      __builtin_amdgcn_sched_barrier(0);
      next = T::mma(a[x], own[x], next);
      if (x + kLead < CK) a[x + kLead] = kread.row(kt, krow, x + kLead);
#pragma unroll
      for (int r = x * kEach; r < 16 && r < (x + 1) * kEach; ++r) {
        s[r] = power<C>(C::MASK == 0 ? __builtin_fmaf(s[r], c, -base) : s[r] - base);
        sum[r & 1] += s[r];
        if (r & 1) p[r >> 3][(r >> 1) & 3] = T::pack(s[r - 1], s[r]);
      }
      asm volatile("" : "+v"(sum[0]), "+v"(sum[1]));
    }
    u32x4 t[2 * TV];
#pragma unroll
    for (int x = 0; x < kLead && x < 2 * TV; ++x) t[x] = vread.transposed(vt, vrow + 16 * (x / TV), x % TV);
    peak = neg_inf();
    constexpr int kMost = (16 + 2 * TV - 1) / (2 * TV);
#pragma unroll
    for (int x = 0; x < 2 * TV; ++x) {
      __builtin_amdgcn_sched_barrier(0);
      acc[x % TV] = T::mma(t[x], p[x / TV], acc[x % TV]);
      if (x + kLead < 2 * TV) t[x + kLead] = vread.transposed(vt, vrow + 16 * ((x + kLead) / TV), (x + kLead) % TV);
#pragma unroll
      for (int r = x * kMost; C::MASK == 0 && r < 16 && r < (x + 1) * kMost; ++r) peak = __builtin_fmaxf(peak, next[r]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (C::MASK != 0 || __any(j0 + 64 > seen)) {
      __builtin_amdgcn_sched_barrier(0);
      peak = limit(j0 + 32, next);
    }
    s = next;
  };
  bool active = first < end && __any(first < seen);   // (wavefronts whose rows see nothing of a tile only help to fetch the next one)
  if (active) {
    if (C::MASK != 0) {
      part = maskRow.part(first, half);
      later = maskRow.part(first + 32, half);
    }
    s = {};
#pragma unroll
    for (int x = 0; x < CK; ++x) s = T::mma(kread.row(ktiles[0], 0, x), own[x], s);
    peak = limit(first, s);
  }
  int buf = 0;
  for (int k0 = first; k0 < end; k0 += kTile) {
    const int next = buf + 1 < kTiles ? buf + 1 : 0, then = kTiles == 2 ? buf : next + 1 < kTiles ? next + 1 : 0;
    fetch(k0 + 2 * kTile < end ? k0 + 2 * kTile : kl);   // (none left: zeros, nothing is asked of memory)
    if (active) {
      step(k0, vtiles[buf], 0, ktiles[buf], 32);
      step(k0 + 32, vtiles[buf], 32, ktiles[next], 0);
      active = k0 + kTile < end && __any(k0 + kTile < seen);
    }
    if (k0 + kTile >= end) break;
    if (kTiles == 2) __syncthreads();   // (the tile written now has been read until here)
    kload.store(ktiles[then], tid);
    vload.store(vtiles[then], tid);
    __syncthreads();
    buf = next;
  }

  const float all = add_halves(sum[0] + sum[1]);
  if (SPLIT) {
    auto &meet = reinterpret_cast<Meeting<kThreads> &>(lds);
    const Ranges<C> ranges(ws, heads * tiles, heads * rows, splits);
    const long slot = head * rows + row;
    if (exists) {
      if (all > 0.0f || all != all) {
#pragma unroll
        for (int d = 0; d < TV; ++d) {
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const float x[4] = {acc[d][4 * r4], acc[d][4 * r4 + 1], acc[d][4 * r4 + 2], acc[d][4 * r4 + 3]};
            ws_store_chunk<4>(ranges.ws, ranges.accumulator(split, slot, 32 * d + 8 * r4 + 4 * half), x);
          }
        }
      }
      const float state[2] = {top, all};
      if (half == 0) ws_store_chunk<2>(ranges.ws, ranges.state(split, slot), state);
    }
    if (!JOIN || !last_workgroup(ranges.counters, id, splits, tid, &meet.flag)) return;
    const long count = rows - row0 < kGroup ? rows - row0 : kGroup;
    join<C, kThreads>(ranges, meet, b, hkv, row0, head * rows + row0, static_cast<int>(count), out, lse, e, tid);
    return;
  }
  if (!exists) return;
  const float inverse = all == 0.0f ? 0.0f : 1.0f / all;
  const RowsOf<C, DV> orows(out, b, hkv, e);
  char *to = const_cast<char *>(orows.base) + orows.offset(row);
#pragma unroll
  for (int d = 0; d < TV; ++d) {
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int at = 32 * d + 8 * r4 + 4 * half;
      if (DV % 32 != 0 && at >= DV) continue;
      u32x2 w;
      w[0] = T::pack(acc[d][4 * r4] * inverse, acc[d][4 * r4 + 1] * inverse);
      w[1] = T::pack(acc[d][4 * r4 + 2] * inverse, acc[d][4 * r4 + 3] * inverse);
      *reinterpret_cast<u32x2 *>(to + 2 * at) = w;
    }
  }
  if (lse != nullptr && half == 0) lse[(b * C::H + hkv * C::G + row % C::G) * e.sq + i] = log_sum<C>(top, all);
}

// ---- backward ---------------------------------------------------------------------------------------------------------
// float16 ends at 65504 and has no digits left below 2^-24, and what the matrix units take as float16 is a probability, at
// most 1 and over a long axis arbitrarily small, and a score's gradient, that probability times a difference with
//   |dp - delta| <= B = sum |dout| max |v| + |delta|   (sums over the row's channels).
// The gradients of the scores are therefore computed times the power of two that puts B into [2^13, 2^14) (dq: B of the row and
// all keys of its key head; dk: the largest of the rows that a workgroup takes and the keys of a wavefront), and the probabilities of dv times 2^13: a probability that float32 puts a little above 1 still
// fits, normal numbers reach down to 2^-27 of the largest. The results are scaled back in float32. (bfloat16 has the
// exponents of float32: factor 1.)
constexpr float kProbabilityLift = 13.0f;   // exponent of 2
template <typename T>
AKG_DEV float lift_of(float bound) {
  if (!T::kNarrowRange || !(bound > 0.0f && bound < __builtin_inff())) return 1.0f;
  return __builtin_ldexpf(1.0f, 14 - __builtin_amdgcn_frexp_expf(bound));   // bound = m 2^exponent, 1/2 <= m < 1; lifts from 2^-27 to 2^62
}
AKG_DEV float max_lanes(float v) {
#pragma unroll
  for (int step = 1; step < 64; step *= 2) v = __builtin_fmaxf(v, __shfl_xor(v, step));
  return v;
}

// What the backward kernels know of a row's sum: exp(score - lse) = 2^((score - top) log2 e - rest), rest = 0 where lse says
// it. Where a mask is added and lse is large (rows whose mask is -1e9 throughout), a float32 lse has lost the log of the
// sum behind the maximum: the kernel of dq then finds both again.
constexpr float kLargeLse = 4096.0f;

// Places in the workspace of the backward kernels, in floats: delta and top of every row (top: times log2 e where no mask is
// added; infinite for a row without keys, whose probabilities then are 2^-inf = 0), for an added mask the rest; for float16
// what bounds the gradients of the scores: the largest sum |dout| and |delta| of every wavefront of the first kernel, and the
// largest |v| of every slice of a key head's keys.
template <typename C>
struct BackwardSpace {
  long rows;         // of all key heads
  long wavefronts;   // of the first kernel, over all key heads
  static constexpr bool kBounds = C::T::kNarrowRange;
  AKG_DEV long top(long row) const { return rows + row; }
  AKG_DEV long rest(long row) const { return 2 * rows + row; }
  AKG_DEV long sizes(long wavefront) const { return (C::ADDED ? 3 : 2) * rows + 2 * wavefront; }
  AKG_DEV long values(long slice) const { return sizes(wavefronts) + slice; }
  // behind them, to the next 256 bytes: sums of dk and dv over ranges of rows, [ranges][key heads][keys][padded channels of both]
  static constexpr int kSums = padded(C::DK) + padded(C::DV);
  AKG_DEV long sums(long heads, long sk) const { return ((kBounds ? values(heads * value_slices(sk)) : sizes(0)) + 63) / 64 * 64; }
  // Slices of a key head's keys, 128 keys each or more.
  AKG_DEV static long value_slices(long sk) { return sk <= 128 * 256 ? (sk + 127) / 128 : 256; }
  // The largest |v| of key head `head`, in every lane.
  AKG_DEV float largest_value(const float *ws, long head, long sk, int lane) const {
    const long slices = value_slices(sk);
    float largest = 0.0f;
    for (long t = lane; t < slices; t += 64) largest = __builtin_fmaxf(largest, ws[values(head * slices + t)]);
    return max_lanes(largest);
  }
};

// The largest |v| of one slice of the keys of a key head, by a workgroup of 256 threads: a launch of its own, or workgroups
// beside those that find what else the rows need, for dq. It reads the values once more: float16 gradients of 8 x 200 x 12 heads of 64
// take 20.4 us with it and 19.4 without, of 1 x 1024 x 16/4 of 128 78 and 75, of 2 x 4096 x 32/8 of 128 983 and 975.
template <typename C>
AKG_DEV void slice_of_values(const void *v, const int *klens, float *ws, Extents e, long wavefronts, long block) {
  typedef typename C::T T;
  __shared__ float tops[4];
  const long heads = e.batch * C::HKV, slices = BackwardSpace<C>::value_slices(e.sk), head = block / slices, slice = block % slices;
  const long b = head / C::HKV, hkv = head % C::HKV, each = (e.sk + slices - 1) / slices;
  const int kl = clamped_length<C>(klens, b, e.sk), tid = static_cast<int>(threadIdx.x);
  const KeysOf<C, C::DV> values(v, b, hkv, e);
  const long first = slice * each, left = kl - first < each ? kl - first : each;
  constexpr int kPerRow = C::DV / 8;
  float largest = 0.0f;
#pragma unroll 4
  for (long c = tid; c < left * kPerRow; c += 256) {
    const u32x4 x = *reinterpret_cast<const u32x4 *>(values.base + (first + c / kPerRow) * values.step + c % kPerRow * 16);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      largest = __builtin_fmaxf(largest, __builtin_fmaxf(__builtin_fabsf(T::low(x[w])), __builtin_fabsf(T::high(x[w]))));
    }
  }
  largest = max_lanes(largest);
  if ((tid & 63) == 0) tops[tid >> 6] = largest;
  __syncthreads();
  if (tid == 0) {
    const BackwardSpace<C> space{heads * e.sq * C::G, wavefronts};
    ws[space.values(head * slices + slice)] = __builtin_fmaxf(__builtin_fmaxf(tops[0], tops[1]), __builtin_fmaxf(tops[2], tops[3]));
  }
}

// dq of 32 rows a wavefront: keys and values pass by in tiles, 32 keys a step: the scores and their gradients' products, then
// the gradients of the scores (vector instructions) between the matrix instructions that multiply those of the step before.
// Leaves in `ws` what the kernel of dk and dv needs. Bound as the forward pass is: the training case there takes 390 to 412 us,
// 1.0 to 1.06 PFLOP/s of its three products, by the card, once that holds its clock, and up to 530 in the milliseconds behind a
// pause (2 % more with the gradients of a step computed in front of its own products).
// PART: 0 all of it; 1 only what it leaves in `ws`; 2 only dq, from that.
template <typename C, int NW, int PART>
struct QueriesLds {
  static constexpr int kTiles = NW == 8 && 3 * kTile * (pitch(C::DK) + pitch(C::DV)) <= 160 * 1024 ? 3 : 2;   // (as in the forward pass)
  __attribute__((aligned(16))) u8 ktiles[kTiles][PART == 1 ? 16 : kTile * pitch(C::DK)], vtiles[kTiles][PART == 1 ? 16 : kTile * pitch(C::DV)];
};
template <typename C, int NW, int PART>
AKG_DEV void backward_queries(const void *dout, const void *q, const void *k, const void *v, const void *out, const float *lse,
                              const void *mask, const int *qlens, const int *klens, void *dq, float *ws, Extents e, float scale, long block,
                              QueriesLds<C, NW, PART> &lds) {
  typedef typename C::T T;
  constexpr int DK = C::DK, DV = C::DV, CK = (DK + 15) / 16, CV = (DV + 15) / 16, TK = padded(DK) / 32, kThreads = 64 * NW;
  constexpr int kTiles = QueriesLds<C, NW, PART>::kTiles;
  auto &ktiles = lds.ktiles;
  auto &vtiles = lds.vtiles;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const long rows = e.sq * C::G, tiles = (rows + kRows * NW - 1) / (kRows * NW), heads = e.batch * C::HKV;
  long head, tile;
  head_and_tile(block, heads, head, tile);
  tile = tiles - 1 - tile;
  const long b = head / C::HKV, hkv = head % C::HKV;
  const int ql = clamped_length<C>(qlens, b, e.sq), kl = clamped_length<C>(klens, b, e.sk);
  const long row0 = tile * (kRows * NW), row = row0 + wave * kRows + (lane & 31);
  const long i = row / C::G, g = row % C::G;
  const bool exists = row < rows;
  const int seen = exists ? keys_seen<C>(i, ql, kl) : 0;
  long last = (row0 + kRows * NW < rows ? row0 + kRows * NW : rows) - 1;
  long lastI = last / C::G;
  if (lastI >= ql) lastI = ql - 1;
  const int end = row0 / C::G < ql ? keys_seen<C>(lastI, ql, kl) : 0;

  const RowsOf<C, DK> qrows(q, b, hkv, e);
  const RowsOf<C, DV> grows(dout, b, hkv, e), orows(out, b, hkv, e);
  u32x4 own[CK], grad[CV];
  load_own<DK>(qrows.base + qrows.offset(exists ? row : 0), seen > 0, lane, own);
  load_own<DV>(grows.base + grows.offset(exists ? row : 0), seen > 0, lane, grad);
  const BackwardSpace<C> space{heads * rows, heads * tiles * NW};
  const float topValue = T::kNarrowRange && PART != 1 ? space.largest_value(ws, head, e.sk, lane) : 0.0f;
  float delta = 0.0f, spread = 0.0f;   // spread: sum |dout|
  {
    u32x4 o[CV] = {};
    if (PART != 2) load_own<DV>(orows.base + orows.offset(exists ? row : 0), seen > 0, lane, o);
#pragma unroll
    for (int x = 0; x < CV; ++x) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (PART != 2) delta = __builtin_fmaf(T::low(o[x][w]), T::low(grad[x][w]), delta);
        if (PART != 2) delta = __builtin_fmaf(T::high(o[x][w]), T::high(grad[x][w]), delta);
        if (T::kNarrowRange) spread += __builtin_fabsf(T::low(grad[x][w])) + __builtin_fabsf(T::high(grad[x][w]));
      }
    }
    delta = add_halves(delta);
  }
  if (PART != 2 && exists && half == 0) ws[head * rows + row] = delta;
  if (PART == 2 && exists) delta = ws[head * rows + row];
  float lift = 1.0f;
  if (T::kNarrowRange) {
    spread = add_halves(spread);
    if (PART != 1) lift = lift_of<T>(__builtin_fmaf(spread, topValue, __builtin_fabsf(delta)));
    if (PART != 2) {
      const float largest = max_lanes(spread), largestDelta = max_lanes(__builtin_fabsf(delta));
      const long at = space.sizes((head * tiles + tile) * NW + wave);
      if (lane == 0) ws[at] = largest;
      if (lane == 0) ws[at + 1] = largestDelta;
    }
  }
  float sums = PART != 2 && exists && seen > 0 ? lse[(b * C::H + hkv * C::G + g) * e.sq + i] : neg_inf();
  // (a row without keys: exp2(s - inf) = 0)
  const bool lost = C::ADDED && __builtin_fabsf(sums) > kLargeLse && __builtin_fabsf(sums) < __builtin_inff();
  sums = sums == neg_inf() ? __builtin_inff() : C::ADDED ? sums : sums * kLog2e;
  float rest = 0.0f;
  if (PART == 2 && exists) sums = ws[space.top(head * rows + row)];
  if (PART == 2 && C::ADDED && exists) rest = ws[space.rest(head * rows + row)];
  const float c = C::ADDED ? scale : scale * kLog2e;

  f32x16 acc[TK];
#pragma unroll
  for (int d = 0; d < TK; ++d) acc[d] = {};
  const KeysOf<C, DK> keys(k, b, hkv, e);
  const KeysOf<C, DV> values(v, b, hkv, e);
  const Reader<DK> kread(lane);
  const Reader<DV> vread(lane);
  TileLoad<kTile, DK, kThreads> kload;
  TileLoad<kTile, DV, kThreads> vload;
  auto fetch = [&](int k0) {
    const Buffer kb = make_buffer(keys.base + k0 * keys.step, records((kl - k0 - 1) * keys.step + 2 * DK));
    const Buffer vb = make_buffer(values.base + k0 * values.step, records((kl - k0 - 1) * values.step + 2 * DV));
    kload.load(kb, tid, [&](int r) { return static_cast<u32>(r * static_cast<int>(keys.step)); });
    vload.load(vb, tid, [&](int r) { return static_cast<u32>(r * static_cast<int>(values.step)); });
  };
#pragma unroll
  for (int x = 0; PART != 1 && x < kTiles; ++x) {
    clear_padding<kTile, DK, kThreads>(ktiles[x], tid);
    clear_padding<kTile, DV, kThreads>(vtiles[x], tid);
  }
  if (PART != 1 && end > 0) {
    fetch(0);
    const TileLoad<kTile, DK, kThreads> know = kload;
    const TileLoad<kTile, DV, kThreads> vnow = vload;
    fetch(kTile < end ? kTile : kl);
    know.store(ktiles[0], tid);
    vnow.store(vtiles[0], tid);
    kload.store(ktiles[1], tid);
    vload.store(vtiles[1], tid);
  }
  __syncthreads();
  const long maskAt = C::MASK != 0 ? mask_row<C>(b, hkv * C::G + g, exists ? i : 0, e) : 0;
  if constexpr (C::ADDED && PART != 2) {
    if (__any(lost)) {   // (by this wavefront alone, keys straight from memory: such rows are rare)
      float top = neg_inf(), sum = 0.0f;
      for (int k0 = 0; __any(k0 < seen); k0 += 32) {
        f32x16 s = {};
        const int key = k0 + (lane & 31);
        u32x4 operand[CK];
        load_own<DK>(keys.base + (key < kl ? key : 0) * keys.step, key < kl, lane, operand);
#pragma unroll
        for (int x = 0; x < CK; ++x) s = T::mma(operand[x], own[x], s);
        float peak = neg_inf();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = k0 + 8 * (r >> 2) + 4 * half + (r & 3);
          s[r] = j < seen ? with_mask<C>(s[r], c, mask, maskAt + j) : neg_inf();
          peak = __builtin_fmaxf(peak, s[r]);
        }
        const float m = __builtin_fmaxf(top, max_halves(peak)), base = m == neg_inf() ? 0.0f : m;
        sum *= power<C>(top - base);
        top = m;
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += power<C>(s[r] - base);
      }
      sum = add_halves(sum);
      if (lost && sum > 0.0f) {
        sums = top;
        rest = __builtin_amdgcn_logf(sum);
      }
    }
    if (exists && half == 0) ws[space.rest(head * rows + row)] = rest;
  }
  if (PART != 2 && exists && half == 0) ws[space.top(head * rows + row)] = sums;
  if (PART == 1) return;
  const MaskRow<C> maskRow(mask, maskAt, e);
  // What the mask says of 32 keys and the next, where registers allow.
  constexpr bool kAhead = padded(DK) + padded(DV) <= 192 || sizeof(typename MaskRow<C>::E) < 4;
  typename MaskRow<C>::Part part, later;
  constexpr int kLead = 4;
  f32x16 s, dp;
  u32x4 ds[2];   // gradients of the scores of 32 keys, rounded (half a step of each, of changing sign)
  // The scores of the keys from j0 on (rows `at` of the tiles) and the products dout v.
  auto scores = [&](int j0, const u8 *kt, const u8 *vt, int at) {
    if (C::MASK != 0) {
      if (kAhead) part = later;
      (kAhead ? later : part) = maskRow.part(kAhead ? j0 + 32 : j0, half);
      if (!kAhead) __builtin_amdgcn_sched_barrier(0);
    }
    s = {};
    dp = {};
    u32x4 a[CK + CV];
    auto operand = [&](auto x) {
      constexpr int m = decltype(x)::value;
      if constexpr (m < CK) {
        return kread.row(kt, at, m);
      } else {
        return vread.row(vt, at, m - CK);
      }
    };
    unrolled<(kLead < CK + CV ? kLead : CK + CV)>([&](auto x) { a[decltype(x)::value] = operand(x); });
    unrolled<CK + CV>([&](auto x) {
      constexpr int m = decltype(x)::value;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (m < CK) {
        s = T::mma(a[m], own[m], s);
      } else {
        dp = T::mma(a[m], grad[m - CK], dp);
      }
      if constexpr (m + kLead < CK + CV) a[m + kLead] = operand(IntTag<m + kLead>());
    });
    __builtin_amdgcn_sched_barrier(0);
    if (C::MASK != 0) maskRow.fix(part, j0, half);
#pragma unroll
    for (int r = 0; C::MASK != 0 && r < 16; ++r) s[r] = part.apply(s[r], c, r);
    if (__any(j0 + 32 > seen)) {
      __builtin_amdgcn_sched_barrier(0);   // (a branch, not a select for every tile)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool ok = j0 + 8 * (r >> 2) + 4 * half + (r & 3) < seen;
        s[r] = ok ? s[r] : neg_inf();
        dp[r] = ok ? dp[r] : 0.0f;
      }
    }
  };
  auto pair = [&](int r, u32x4 (&to)[2]) {
    float y[2];
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      float x = C::MASK != 0 ? s[r + o] - sums : __builtin_fmaf(s[r + o], c, -sums);
      if (C::ADDED) x = __builtin_fmaf(x, kLog2e, -rest);
      y[o] = __builtin_amdgcn_exp2f(x) * (T::kNarrowRange ? (dp[r + o] - delta) * lift : dp[r + o] - delta);
    }
    u32 w = T::pack(y[0], y[1]);
    asm volatile("" : "+v"(w));   // (computed here: left to itself the compiler moves it behind the matrix instructions)
    to[r >> 3][(r >> 1) & 3] = w;
  };
  // The products of the step before (rows `at` of `kt`), and between them the gradients of the scores of this one (of whatever
  // is there behind the last step: one stream without branches, or the accumulators are held twice).
  auto products = [&](const u8 *kt, int at) {
    u32x4 a[2 * TK], to[2];
    auto operand = [&](int m) { return kread.transposed(kt, at + 16 * (m / TK), m % TK); };
    unrolled<(kLead < 2 * TK ? kLead : 2 * TK)>([&](auto x) { a[decltype(x)::value] = operand(decltype(x)::value); });
    unrolled<2 * TK>([&](auto x) {
      constexpr int m = decltype(x)::value;
      __builtin_amdgcn_sched_barrier(0);
      acc[m % TK] = T::mma(a[m], ds[m / TK], acc[m % TK]);
      if constexpr (m + kLead < 2 * TK) a[m + kLead] = operand(m + kLead);
      constexpr int from = m * 8 / (2 * TK), count = (m + 1) * 8 / (2 * TK) - from;   // of eight pairs
      unrolled<count>([&](auto y) { pair(2 * (from + decltype(y)::value), to); });
    });
    __builtin_amdgcn_sched_barrier(0);
    ds[0] = to[0];
    ds[1] = to[1];
  };
  bool active = end > 0 && __any(0 < seen);   // (wavefronts whose rows see nothing of a tile only help to fetch the next one)
  if (active) {
    if (C::MASK != 0 && kAhead) later = maskRow.part(0, half);
    scores(0, ktiles[0], vtiles[0], 0);
    unrolled<8>([&](auto y) { pair(2 * decltype(y)::value, ds); });
  }
  int buf = 0;
  for (int k0 = 0; k0 < end; k0 += kTile) {
    const int next = buf + 1 < kTiles ? buf + 1 : 0, then = kTiles == 2 ? buf : next + 1 < kTiles ? next + 1 : 0;
    fetch(k0 + 2 * kTile < end ? k0 + 2 * kTile : kl);   // (none left: zeros, nothing is asked of memory)
    if (active) {
      scores(k0 + 32, ktiles[buf], vtiles[buf], 32);
      products(ktiles[buf], 0);
      scores(k0 + kTile, ktiles[next], vtiles[next], 0);
      products(ktiles[buf], 32);
      active = __any(k0 + kTile < seen);
    }
    if (k0 + kTile >= end) break;
    if (kTiles == 2) __syncthreads();   // (the tile written now has been read until here)
    kload.store(ktiles[then], tid);
    vload.store(vtiles[then], tid);
    __syncthreads();
    buf = next;
  }
  if (!exists) return;
  const float back = scale / lift;
  const RowsOf<C, DK> drows(dq, b, hkv, e);
  char *to = const_cast<char *>(drows.base) + drows.offset(row);
#pragma unroll
  for (int d = 0; d < TK; ++d) {
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int at = 32 * d + 8 * r4 + 4 * half;
      if (DK % 32 != 0 && at >= DK) continue;
      u32x2 w;
      w[0] = T::pack(acc[d][4 * r4] * back, acc[d][4 * r4 + 1] * back);
      w[1] = T::pack(acc[d][4 * r4 + 2] * back, acc[d][4 * r4 + 3] * back);
      *reinterpret_cast<u32x2 *>(to + 2 * at) = w;
    }
  }
}

// dk and dv of 32 keys a wavefront: the queries of all heads that share them pass by in tiles. RG groups of wavefronts have
// the same keys and take the tiles of rows in turns; their sums are joined at the end, in LDS. (Causal: the first keys are
// seen by all rows, and a workgroup that goes through them alone is the last to end.)
// SPLIT: where the tiles of keys are fewer than the CUs, `splits` workgroups take a range of the rows each and leave their
// sums in `ws` for backward_join. Two groups of wavefronts hide each other's vector instructions behind matrix instructions:
// the training case of the forward pass takes 520 to 557 us, 0.99 to 1.06 PFLOP/s of its four products, by the card, once
// that holds its clock (the whole gradient 918 us, with one group 1074).
// APART: above 256 channels (keys and values together) the accumulators of both leave too little room for the operands: a
// workgroup computes dk or dv, and the scores are computed twice (gradient of 2 x 2048, 32/8 heads of 256, causal: 952 us
// instead of 2423; of 192: 770 instead of 809).
// WHICH: 0 both (or, APART, one a workgroup), 1 dk, 2 dv.
template <typename C, int NW, int RG>
struct KeysLds {
  // From 192 channels on (keys and values together) the accumulators and the wavefront's own operands would leave room for
  // one wavefront per SIMD: its keys lie in LDS then, and two fit.
  static constexpr bool kKeysInLds = padded(C::DK) + padded(C::DV) > 192;
  static constexpr int kRound = kTileRows * RG, kStates = C::ADDED ? 3 : 2;   // states of a row: delta, top and rest (BackwardSpace)
  __attribute__((aligned(16))) u8 rows[2][kRound * (pitch(C::DK) + pitch(C::DV))];
  __attribute__((aligned(16))) u8 own[kKeysInLds ? kRows * NW * own_pitch(C::DK) : 16];
  __attribute__((aligned(16))) float states[2][kStates][kRound];
};
template <typename C, int NW, int RG, int NWQ, bool SPLIT, bool APART, int WHICH>
AKG_DEV void backward_keys(const void *dout, const void *q, const void *k, const void *v, const void *mask,
                           const int *qlens, const int *klens, void *dk, void *dv, float *ws, Extents e, float scale, int splits, long blockId, KeysLds<C, NW, RG> &memory) {
  typedef typename C::T T;
  constexpr int DK = C::DK, DV = C::DV, CK = (DK + 15) / 16, CV = (DV + 15) / 16, TK = padded(DK) / 32, TV = padded(DV) / 32, kThreads = 64 * NW * RG, kRound = kTileRows * RG;
  typedef KeysLds<C, NW, RG> Memory;
  constexpr bool kKeysInLds = Memory::kKeysInLds;
  constexpr int kStates = Memory::kStates;
  auto &lds = memory.rows;
  auto &ownKeys = memory.own;
  auto &stateOf = memory.states;
  auto run = [&](auto which) __attribute__((always_inline)) {
    constexpr bool kDk = decltype(which)::value != 2, kDv = decltype(which)::value != 1;
    const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NW, group = __builtin_amdgcn_readfirstlane(tid >> 6) / NW, half = lane >> 5;
    const long rows = e.sq * C::G, heads = e.batch * C::HKV;
    const long block = APART ? blockId / 2 : blockId, id = SPLIT ? block / splits : block;
    const int split = SPLIT ? static_cast<int>(block % splits) : 0;
    long head, tile;
    head_and_tile(id, heads, head, tile);
    // (the first keys are seen by most queries, and come first)
    const long b = head / C::HKV, hkv = head % C::HKV;
    const int ql = clamped_length<C>(qlens, b, e.sq), kl = clamped_length<C>(klens, b, e.sk);
    const int key0 = static_cast<int>(tile) * (kRows * NW) + wave * kRows;
    const int key = key0 + (lane & 31);
    const bool counts = key < kl;
    const KeysOf<C, DK> keys(k, b, hkv, e);
    const KeysOf<C, DV> values(v, b, hkv, e);
    const long wavesQ = (rows + kRows * NWQ - 1) / (kRows * NWQ) * NWQ;
    const BackwardSpace<C> space{heads * rows, heads * wavesQ};
    u32x4 own[kKeysInLds ? 1 : CK], val[CV] = {};
    if constexpr (kKeysInLds) {
      const int key00 = static_cast<int>(tile) * (kRows * NW);
      const Buffer kb = make_buffer(keys.base + key00 * keys.step, records((kl - key00 - 1) * keys.step + 2 * DK));
      TileLoad<kRows * NW, DK, kThreads> kload;
      kload.load(kb, tid, [&](int r) { return static_cast<u32>(r * static_cast<int>(keys.step)); });
      kload.template store<true>(ownKeys, tid);   // (padding channels meet zeros of the queries, but must be finite)
      for (int c = tid; DK % 32 != 0 && c < kRows * NW * ((padded(DK) - DK) / 8); c += kThreads) {
        constexpr int kPad = DK % 32 != 0 ? (padded(DK) - DK) / 8 : 1;
        *reinterpret_cast<u32x4 *>(ownKeys + c / kPad * own_pitch(DK) + (DK / 8 + c % kPad) * 16) = u32x4{0, 0, 0, 0};
      }
    } else {
      load_own<DK>(keys.base + (counts ? key : 0) * keys.step, counts, lane, own);
    }
    if (kDk) load_own<DV>(values.base + (counts ? key : 0) * values.step, counts, lane, val);
    const float c = C::ADDED ? scale : scale * kLog2e;
    f32x16 acck[kDk ? TK : 1], accv[kDv ? TV : 1];
#pragma unroll
    for (int d = 0; kDk && d < TK; ++d) acck[d] = {};
#pragma unroll
    for (int d = 0; kDv && d < TV; ++d) accv[d] = {};

    // queries that see the first key of the workgroup, up to the last one of the sequence
    const int first0 = static_cast<int>(tile) * (kRows * NW);
    int from = 0;
    if (C::CAUSAL) {
      const long i = static_cast<long>(first0) - kl + ql;
      from = static_cast<int>((i > 0 ? (i < ql ? i : ql) : 0) * C::G / kRound * kRound);
    }
    int upto = first0 < kl ? ql * C::G : 0;
    if (SPLIT && from < upto) {
      const int rounds = (upto - from + kRound - 1) / kRound, each = (rounds + splits - 1) / splits * kRound;
      const long start = from + static_cast<long>(split) * each;
      from = start < upto ? static_cast<int>(start) : upto;
      if (each < upto - from) upto = from + each;
    }

    // (of the rows that this workgroup takes and the wavefront's own keys: what others have costs these no digits)
    float lift = 1.0f;
    if (kDk && T::kNarrowRange) {
      float largest = 0.0f, largestDelta = 0.0f, largestValue = 0.0f;
#pragma unroll
      for (int x = 0; x < CV; ++x) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          largestValue = __builtin_fmaxf(largestValue, __builtin_fmaxf(__builtin_fabsf(T::low(val[x][w])), __builtin_fabsf(T::high(val[x][w]))));
        }
      }
      for (long t = from / kRows + lane; t * kRows < upto; t += 64) {
        const long at = space.sizes(head * wavesQ + t);
        largest = __builtin_fmaxf(largest, ws[at]);
        largestDelta = __builtin_fmaxf(largestDelta, ws[at + 1]);
      }
      lift = lift_of<T>(__builtin_fmaf(max_lanes(largest), max_lanes(largestValue), max_lanes(largestDelta)));
    }
    // probabilities leave their exponential lifted: the gradients of the scores take that out of their own factor
    constexpr float kLift = T::kNarrowRange ? kProbabilityLift : 0.0f, kUnlift = T::kNarrowRange ? 0x1p-13f : 1.0f;
    const float liftBehind = lift * kUnlift;

    const RowsOf<C, DK> qrows(q, b, hkv, e);
    const RowsOf<C, DV> grows(dout, b, hkv, e);
    const Reader<DK> qread(lane);
    const Reader<DV> gread(lane);
    TileLoad<kRound, DK, kThreads> qload;
    TileLoad<kRound, DV, kThreads> gload;
    // Rows behind the last one read zeros (nothing is asked of memory): their probabilities are 1 (lifted), their products 0.
    float state[kStates];
    auto fetch = [&](int r0, bool any) {
      const int i0 = r0 / C::G;
      const Buffer qb = make_buffer(qrows.base + i0 * qrows.stepI, 0x7fffffffL);
      const Buffer gb = make_buffer(grows.base + i0 * grows.stepI, 0x7fffffffL);
      const int left = any ? upto - r0 : 0, lead = r0 - i0 * C::G;
      auto offsetIn = [&](const auto &of, int r) {
        const int at = lead + r;
        return r < left ? static_cast<u32>(at / C::G * static_cast<int>(of.stepI) + at % C::G * static_cast<int>(of.stepG)) : kBeyondEveryBuffer;
      };
      qload.load(qb, tid, [&](int r) { return offsetIn(qrows, r); });
      gload.load(gb, tid, [&](int r) { return offsetIn(grows, r); });
      if (tid < kRound) {
#pragma unroll
        for (int x = 0; x < kStates; ++x) state[x] = tid < left ? ws[x * heads * rows + head * rows + r0 + tid] : 0.0f;
      }
    };
    auto put = [&](int buf) {
      qload.store(lds[buf], tid);
      gload.store(lds[buf] + kRound * pitch(DK), tid);
      if (tid < kRound) {
#pragma unroll
        for (int x = 0; x < kStates; ++x) stateOf[buf][x][tid] = x == kStates - 1 ? state[x] - kLift : state[x];
      }
    };
#pragma unroll
    for (int buf = 0; buf < 2; ++buf) {
      clear_padding<kRound, DK, kThreads>(lds[buf], tid);
      clear_padding<kRound, DV, kThreads>(lds[buf] + kRound * pitch(DK), tid);
    }
    // The last rows first: all tiles of a key head then pass the same rows at the same time, whatever row their first is, and
    // find them in the L2 (2 x 4096, 32/8 heads of 128, causal: 0.46 GB from memory; the first rows first 1.7 GB, 10 us more).
    const int start = from + (upto - from - 1) / kRound * kRound;
    if (from < upto) {
      fetch(start, true);
      put(0);
    }
    __syncthreads();
    int buf = 0;
    for (int round = start; from < upto && round >= from; round -= kRound, buf ^= 1) {
      const int r0 = round + group * kTileRows, at0 = group * kTileRows;   // this group's tile
      const u8 *qt = lds[buf] + at0 * pitch(DK), *gt = lds[buf] + kRound * pitch(DK) + at0 * pitch(DV);
      // the tile's last row sees most keys, its first one least
      const int lastRow = (r0 + kTileRows < upto ? r0 + kTileRows : upto) - 1;
      const bool active = r0 < upto && key0 < keys_seen<C>(lastRow / C::G, ql, kl);
      u32x4 p[2], ds[2];
      if (active) {
        f32x16 s = {}, dp = {};
        // (what the mask says is asked for before the scores are computed)
        typename MaskRow<C>::E said[16];
        if (C::MASK != 0) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int x = r0 + 8 * (r >> 2) + 4 * half + (r & 3), at = x < upto ? x : upto - 1;
            said[r] = static_cast<const typename MaskRow<C>::E *>(mask)[mask_row<C>(b, hkv * C::G + at % C::G, at / C::G, e) + (counts ? key : 0)];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int x = 0; x < CK; ++x) s = T::mma(qread.row(qt, 0, x), kKeysInLds ? read_own<DK>(ownKeys, wave * kRows, x, lane) : own[kKeysInLds ? 0 : x], s);
#pragma unroll
        for (int x = 0; kDk && x < CV; ++x) dp = T::mma(gread.row(gt, 0, x), val[x], dp);
        FeedOrder<CK + (kDk ? CV : 0), (kKeysInLds ? 2 : 1) * CK + (kDk ? CV : 0), 6>::emit();
        if (C::MASK != 0 || key0 + kRows > keys_seen<C>(r0 / C::G, ql, kl)) {
          __builtin_amdgcn_sched_barrier(0);   // (a branch, not a select for every tile)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at = r0 + 8 * (r >> 2) + 4 * half + (r & 3), i = at / C::G;
            const bool ok = key < keys_seen<C>(i, ql, kl);
            if (C::MASK != 0) {
              s[r] = ok ? with_mask<C>(s[r], c, said, r) : neg_inf();
            } else {
              s[r] = ok ? s[r] : neg_inf();
            }
          }
        }
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 d4 = *reinterpret_cast<const f32x4 *>(&stateOf[buf][0][at0 + 8 * r4 + 4 * half]);
          const f32x4 l4 = *reinterpret_cast<const f32x4 *>(&stateOf[buf][1][at0 + 8 * r4 + 4 * half]);
          f32x4 o4 = {};
          if (C::ADDED) o4 = *reinterpret_cast<const f32x4 *>(&stateOf[buf][kStates - 1][at0 + 8 * r4 + 4 * half]);
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            const int r = 4 * r4 + z;
            float x = C::MASK != 0 ? s[r] - l4[z] : __builtin_fmaf(s[r], c, -l4[z]);
            if (C::ADDED) x = __builtin_fmaf(x, kLog2e, -o4[z]);
            s[r] = __builtin_amdgcn_exp2f(x);
            if (kDk) dp[r] = s[r] * (T::kNarrowRange ? (dp[r] - d4[z]) * liftBehind : dp[r] - d4[z]);
          }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            p[x][w] = T::pack(s[8 * x + 2 * w], s[8 * x + 2 * w + 1]);
            ds[x][w] = T::pack(dp[8 * x + 2 * w], dp[8 * x + 2 * w + 1]);
          }
          asm volatile("" : "+v"(p[x]), "+v"(ds[x]));   // (the scores end here: their registers hold the next tile's rows)
        }
      }
      fetch(round > from ? round - kRound : from, round > from);   // (none left: zeros, nothing is asked of memory)
      if (active) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int d = 0; kDv && d < TV; ++d) accv[d] = T::mma(gread.transposed(gt, 16 * x, d), p[x], accv[d]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int d = 0; kDk && d < TK; ++d) acck[d] = T::mma(qread.transposed(qt, 16 * x, d), ds[x], acck[d]);
        }
        FeedOrder<2 * ((kDv ? TV : 0) + (kDk ? TK : 0)), 4 * ((kDv ? TV : 0) + (kDk ? TK : 0)), 8>::emit();
      }
      put(buf ^ 1);
      __syncthreads();
    }
    // the groups' sums joined: group g leaves as many accumulators as fit where the tiles were, group 0 adds them
    if constexpr (RG > 1) {
      constexpr int kFit = static_cast<int>(sizeof(lds)) / (64 * NW * (RG - 1) * 16), kFoursK = kDk ? 4 * TK : 0, kFours = kFoursK + (kDv ? 4 * TV : 0), kPart = kFit < kFours ? kFit : kFours;
      f32x4 *parts = reinterpret_cast<f32x4 *>(&lds[0][0]);
      unrolled<(kFours + kPart - 1) / kPart>([&](auto pass) {
        constexpr int p0 = decltype(pass)::value * kPart, kCount = kFours - p0 < kPart ? kFours - p0 : kPart;
        __syncthreads();
        if (group > 0) {
          unrolled<kCount>([&](auto y) {
            constexpr int x = p0 + decltype(y)::value, r = 4 * (x % 4);
            const f32x16 &acc = x < kFoursK ? acck[x < kFoursK ? x / 4 : 0] : accv[x < kFoursK ? 0 : (x - kFoursK) / 4];
            parts[(((group - 1) * kPart + x - p0) * NW + wave) * 64 + lane] = f32x4{acc[r], acc[r + 1], acc[r + 2], acc[r + 3]};
          });
        }
        __syncthreads();
        if (group == 0) {
          unrolled<kCount>([&](auto y) {
            constexpr int x = p0 + decltype(y)::value, r = 4 * (x % 4);
            f32x16 &acc = x < kFoursK ? acck[x < kFoursK ? x / 4 : 0] : accv[x < kFoursK ? 0 : (x - kFoursK) / 4];
#pragma unroll
            for (int g = 0; g < RG - 1; ++g) {
              const f32x4 more = parts[((g * kPart + x - p0) * NW + wave) * 64 + lane];
#pragma unroll
              for (int z = 0; z < 4; ++z) acc[r + z] += more[z];
            }
          });
        }
      });
      if (group > 0) return;
    }
    if (key >= e.sk) return;
    const float back = scale / lift;
    if constexpr (SPLIT) {
      float *to = ws + space.sums(heads, e.sk) + ((split * heads + head) * e.sk + key) * BackwardSpace<C>::kSums;
#pragma unroll
      for (int d = kDk ? 0 : TK; d < (kDv ? TK + TV : TK); ++d) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          f32x4 x;
#pragma unroll
          for (int z = 0; z < 4; ++z) x[z] = d < TK ? acck[kDk ? d % TK : 0][4 * r4 + z] * back : accv[kDv && d >= TK ? d - TK : 0][4 * r4 + z] * kUnlift;
          *reinterpret_cast<f32x4 *>(to + 32 * d + 8 * r4 + 4 * half) = x;
        }
      }
      return;
    }
    auto store = [&](char *to, int dim, const f32x16 *acc, int tilesD, float factor) {
#pragma unroll
      for (int d = 0; d < tilesD; ++d) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int at = 32 * d + 8 * r4 + 4 * half;
          if (dim % 32 != 0 && at >= dim) continue;
          u32x2 w;
          w[0] = T::pack(acc[d][4 * r4] * factor, acc[d][4 * r4 + 1] * factor);
          w[1] = T::pack(acc[d][4 * r4 + 2] * factor, acc[d][4 * r4 + 3] * factor);
          *reinterpret_cast<u32x2 *>(to + 2 * at) = w;
        }
      }
    };
    const KeysOf<C, DK> dkeys(dk, b, hkv, e);
    const KeysOf<C, DV> dvalues(dv, b, hkv, e);
    if (kDk) store(const_cast<char *>(dkeys.base) + key * dkeys.step, DK, acck, TK, back);
    if (kDv) store(const_cast<char *>(dvalues.base) + key * dvalues.step, DV, accv, TV, kUnlift);
  };
  if constexpr (APART) {
    if (blockId % 2 == 0) {
      run(IntTag<1>());
    } else {
      run(IntTag<2>());
    }
  } else {
    run(IntTag<WHICH>());
  }
}

// dk and dv from the sums over ranges of rows, in their order: four channels a thread.
template <typename C, int NWQ, int WHICH>
AKG_DEV void backward_join(const float *ws, void *dk, void *dv, Extents e, int splits) {
  typedef typename C::T T;
  constexpr int DK = WHICH != 2 ? C::DK : 0, DV = WHICH != 1 ? C::DV : 0, kFours = (DK + DV) / 4, kSums = BackwardSpace<C>::kSums;
  const long rows = e.sq * C::G, heads = e.batch * C::HKV, wavesQ = (rows + kRows * NWQ - 1) / (kRows * NWQ) * NWQ;
  const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x, row = at / kFours;
  if (row >= heads * e.sk) return;
  const int c = static_cast<int>(at % kFours) * 4;
  const bool isK = c < DK;
  const float *from = ws + BackwardSpace<C>{heads * rows, heads * wavesQ}.sums(heads, e.sk) + row * kSums + (isK ? c : padded(C::DK) + c - DK);
  f32x4 sum = {};
  for (int s = 0; s < splits; ++s) sum += *reinterpret_cast<const f32x4 *>(from + s * heads * e.sk * kSums);
  const long head = row / e.sk, key = row % e.sk, b = head / C::HKV, hkv = head % C::HKV;
  const KeysOf<C, C::DK> dkeys(dk, b, hkv, e);
  const KeysOf<C, C::DV> dvalues(dv, b, hkv, e);
  char *to = isK ? const_cast<char *>(dkeys.base) + key * dkeys.step + 2 * c : const_cast<char *>(dvalues.base) + key * dvalues.step + 2 * (c - DK);
  *reinterpret_cast<u32x2 *>(to) = u32x2{T::pack(sum[0], sum[1]), T::pack(sum[2], sum[3])};
}

}  // namespace attn
}  // namespace akg
