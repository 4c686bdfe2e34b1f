/**
 * Linear attention with a decay for each head, for gfx950. The state of a head is a matrix, keys by values, in float32:
 *
 *   S[t] = exp(g) S[t-1] + k[t] v[t]^T,   out[t] = scale q[t] S[t]
 *
 * A walk over tokens takes a chunk of them at a time, S being the state in front of the chunk (r, c: tokens inside it):
 *
 *   out[r] = scale ( exp(g (r + 1)) q[r] S + sum_{c <= r} exp(g (r - c)) (q[r] . k[c]) v[c] )
 *   S     <- exp(g n) S + sum_c exp(g (n - 1 - c)) k[c] v[c]^T        (n: tokens of the chunk)
 *
 * No exponent is positive where g is not, so nothing overflows however long the walk is. Where g is positive, weights of distances that
 * no two tokens of a walk have are 0 (rows of a tile without a token would meet infinity otherwise), and a state of 0 stays 0. The
 * gradient is three walks of the same form, with dS[t] = scale q[t] dout[t]^T + exp(g) dS[t+1]:
 *
 *   dq[t] = scale dout[t] S[t]^T   (dout, v, k), dk[t] = v[t] dS[t]^T   (v, dout, q) backward, dv[t] = k[t] dS[t]   (k, q, dout) backward
 *
 * so the kernel is written for (a, b, c) -> out with a state of b by c, forward or backward in time (a backward walk
 * numbers the tokens from the last one on). A state that a backward walk is given is that of its first token already: there
 * the exponents of what comes from outside the chunk are one less, and those of what goes on one more.
 *
 * Products run on v_mfma_f32_32x32x16_bf16 with float32 accumulators. A wavefront owns 32 columns of the state (channels
 * of c) as accumulators: what one matrix instruction leaves in a lane is, rounded, the operand of the next one, so the
 * state never leaves the registers. Two quads of channels change places in the transposing LDS reads for that: lane m of a
 * transposed operand holds channel m with bits 2 and 3 swapped, so the rows that a lane holds of a result are eight
 * adjacent channels (the contracted ones of the next product, read from LDS as 16 bytes, and 16 bytes of a row of `out`).
 * The wavefronts share the masked products of a chunk (a . b) through LDS, in the form of the operand that they become.
 *
 * Rounding: bfloat16 operands are exact; products a . b and the state are rounded to bfloat16 (2^-8 of each term at most) where they
 * are contracted again. What is added to the state, exp(g ..) c, goes as two bfloat16 parts (2^-16 of it), since a state gathers what
 * thousands of tokens add, and as three (2^-24) where the last state is a result, in float32. float16 operands, and everything
 * contracted with them, go as two bfloat16 parts throughout: three products for one, no range but that of float32, and 2^-16 of each
 * term.
 *
 * What bounds it: a wavefront that holds a state issues a vector instruction every 5.2 cycles, a matrix instruction of its own every
 * 33, and has 340 of the first (the state rounded and faded, c weighed and split) and 54 of the second for 64 tokens of 128
 * channels; all CUs at work, the clock falls to 1.5 GHz. 4 x 4096 tokens of 32 heads of 128 take 128 us, 4.2 TB/s, 16 x 4096 441 us,
 * 4.9 TB/s; the gradient of the first 303 us for seven tensors, of which it moves ten. (c weighed by the wavefronts that fetch, and
 * read from LDS in parts: a gradient of 2 x 1021 tokens of 16/4 heads 41 us instead of 45, of 4 x 4096 of 32 heads 356 instead of 312,
 * since four wavefronts' tiles then have 32 tokens.)
 */
#pragma once

namespace akg {
namespace linear {

using attn::BF16;
using attn::f32x16;
using attn::f32x4;
using attn::kLog2e;
using attn::padded;
using attn::records;
using attn::u32x2;
using attn::u32x4;

// A tile of W channels in LDS: rows of 64, 128, 256 or 512 bytes without any between them, whose chunks of 16 bytes change places
// by exclusive or with bits of the row. Four neighbouring rows of 64 bytes (transposed reads, half a wavefront at a time) and
// sixteen of 16 bytes (rows read by 128 bits) then lie in banks of their own. The places of a lane differ by an exclusive or with
// a constant. (With 32 and 64 bytes more a row instead, transposed reads met in the banks, or three chunks' tiles did not fit; a
// gradient of 4 x 4096 tokens of 8 heads of 256 took 334 us instead of 242.)
constexpr int pitch(int w) { return w <= 32 ? 64 : w <= 64 ? 128 : w <= 128 ? 256 : 512; }
constexpr int turn(int w, int row) { return (w <= 32 ? 0 : w <= 64 ? (row & 2) << 1 : (row & 3) << 2) | ((row >> 2) & 3); }
// (above 128 channels two wavefronts may share the rows of a state: a multiple of 64)
constexpr int whole(int w) { return w <= 128 ? padded(w) : (w + 63) / 64 * 64; }
template <int W>
AKG_DEV int chunk_at(int row, int chunk) {
  return row * pitch(W) + ((chunk ^ turn(W, row)) << 4);
}
// The channels behind W of a tile's rows, up to whole(W), hold zeros: written once, never again.
template <int ROWS, int W, int THREADS>
AKG_DEV void clear_padding(u8 *tile, int tid) {
  if constexpr (whole(W) != W) {
    constexpr int kPad = (whole(W) - W) / 8;
    for (int c = tid; c < ROWS * kPad; c += THREADS) *reinterpret_cast<u32x4 *>(tile + chunk_at<W>(c / kPad, W / 8 + c % kPad)) = u32x4{0, 0, 0, 0};
  }
}

// Channel of a 32-channel unit that lane `m` (mod 32) of a transposed operand holds.
constexpr int swapped(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

// exp(g n) from g log2 e: 1 for n = 0 (also where g is -inf).
AKG_DEV float power(float g2, int n) { return n == 0 ? 1.0f : __builtin_amdgcn_exp2f(g2 * static_cast<float>(n)); }
// What a state fades by with every chunk: exp(g n) as `whole`, a float32 number, and `rest`, what that leaves of it near 1. A factor
// that is rounded once is off by the same share every time, over 256 chunks by 2^-17; so each chunk's is rounded with what is
// `owed` since the first, and their product stays within a step of float32. (A state faded by s + s (exp(g n) - 1) does not
// drift either, but is off by half a step of what it was, not of what is left of it: with exp(g n) of 2^-24 by all of that.)
struct Fade {
  float whole, rest, owed = 0.0f;
  AKG_DEV void set(float g, int n) {
    const float x = g * static_cast<float>(n);
    rest = 0.0f;
    if (n == 0) {
      whole = 1.0f;
    } else if (!(__builtin_fabsf(x) < 0.125f)) {
      whole = __builtin_amdgcn_exp2f(x * kLog2e);
    } else {
      float p = __builtin_fmaf(x, 1.0f / 720.0f, 1.0f / 120.0f);   // exp(x) - 1: x^7 / 7! is below 2^-30 x there
      p = __builtin_fmaf(x, p, 1.0f / 24.0f);
      p = __builtin_fmaf(x, p, 1.0f / 6.0f);
      p = __builtin_fmaf(x, p, 0.5f);
      p = __builtin_fmaf(x * x, p, x);
      whole = 1.0f + p;
      rest = p - (whole - 1.0f);
    }
  }
  AKG_DEV float next() {
    owed += rest;
    const float f = whole + owed;
    owed -= f - whole;
    return f;
  }
};

// Float32 values as PARTS values of bfloat16 whose sum they are, to 2^-8, 2^-16 or 2^-24 of them: word `e` of an operand.
template <int PARTS>
AKG_DEV void split_pair(float lo, float hi, u32x4 (&parts)[PARTS], int e) {
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    u32 w = BF16::pack(lo, hi);
    if (p + 1 < PARTS) {
      asm("" : "+v"(w));   // (one rounding, not another one for the rest)
      lo -= BF16::low(w);
      hi -= BF16::high(w);
    }
    parts[p][e] = w;
  }
}
template <int PARTS>
AKG_DEV void split(const float (&x)[8], u32x4 (&parts)[PARTS]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) split_pair<PARTS>(x[2 * e], x[2 * e + 1], parts, e);
}

// c += a b, both in parts (the product of the two rests is below every digit kept).
template <int PA, int PB>
AKG_DEV f32x16 product(const u32x4 (&a)[PA], const u32x4 (&b)[PB], f32x16 c) {
  if constexpr (PB == 2) c = BF16::mma(a[0], b[1], c);
  if constexpr (PA == 2) c = BF16::mma(a[1], b[0], c);
  return BF16::mma(a[0], b[0], c);
}

// A lane's places in a tile of W channels (as attn::Reader, with the quads of transposed reads swapped). A tile lies `tile` bytes
// behind `lds`, both multiples of 256.
template <int W>
struct Places {
  int along, across[2];
  AKG_DEV explicit Places(int lane) {
    const int h = lane >> 5, i = lane & 15, r = 4 * h + (i >> 2), quad = ((i & 1) << 1) | ((i & 2) >> 1), chunk = 2 * ((lane >> 4) & 1) + (quad >> 1);
    along = chunk_at<W>(lane & 31, h);
    across[0] = chunk_at<W>(r, chunk) + (quad & 1) * 8;
    across[1] = chunk_at<W>(r + 8, chunk) + (quad & 1) * 8;
  }
  // Channels 16 c + 8 (lane / 32) .. + 7 of row `row0 + lane % 32` (row0 a multiple of 32).
  AKG_DEV u32x4 row(const u8 *lds, int tile, int row0, int c) const {
    return *reinterpret_cast<const u32x4 *>(lds + ((tile + along) ^ (32 * c)) + row0 * pitch(W));
  }
  // Channel 32 unit + swapped(lane % 32) of the rows row0 + 4 h .. 4 h + 3 and row0 + 8 + 4 h .. (h = lane / 32; row0 a multiple of 16).
  AKG_DEV u32x4 transposed(const u8 *lds, int tile, int row0, int unit) const {
    const attn::s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attn::s16x4 *)(lds + ((tile + across[0]) ^ (64 * unit)) + row0 * pitch(W)));
    const attn::s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) attn::s16x4 *)(lds + ((tile + across[1]) ^ (64 * unit)) + row0 * pitch(W)));
    const u32x2 l = __builtin_bit_cast(u32x2, lo), u = __builtin_bit_cast(u32x2, hi);
    return u32x4{l[0], l[1], u[0], u[1]};
  }
};

// The last `count` of the rows of a tile in memory: row ROWS - 1 - i is i (BACK) or count - 1 - i rows behind `first`; `channels`
// of a row are read.
template <int ROWS, bool BACK>
struct Rows {
  Buffer buf;
  int from, each, missing, channels;
  AKG_DEV Rows(const char *first, long step, int count, int channels_)
      : buf(make_buffer(first, count > 0 ? records((count - 1) * step + 2L * channels_) : 0)), from((BACK ? ROWS - 1 : count - ROWS) * static_cast<int>(step)),
        each(BACK ? -static_cast<int>(step) : static_cast<int>(step)), missing(ROWS - count), channels(channels_) {}
};
// ROWS tokens of W channels on their way from memory to LDS, in kEach pieces of a thread. Tokens and channels that do not exist
// read zeros.
template <int ROWS, int W, int THREADS, int PARTS>
struct Stage {
  static constexpr int kPerRow = W / 8, kChunks = ROWS * kPerRow, kEach = (kChunks + THREADS - 1) / THREADS;
  static constexpr bool kWhole = kChunks % THREADS == 0;
  // (the rows of a thread then lie a constant number of rows apart, at the same place of their swizzle)
  static constexpr bool kEven = kWhole && THREADS % kPerRow == 0 && THREADS / kPerRow % 16 == 0;
  static constexpr int kTileBytes = ROWS * pitch(W);
  static constexpr u32 kInfinity = PARTS == 1 ? 0x7f80 : 0x7c00;   // of bfloat16, float16
  u32x4 held[kEach];
  template <bool BACK>
  AKG_DEV void load(const Rows<ROWS, BACK> &rows, int i, int tid) {
    const int c = tid + i * THREADS, row = c / kPerRow, at = c % kPerRow * 8;
    const bool there = row >= rows.missing && at < rows.channels && (kWhole || c < kChunks);
    held[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows.buf, there ? static_cast<u32>(rows.from + row * rows.each + 2 * at) : kBeyondEveryBuffer, 0, 0));
  }
  // Whether a piece of this thread holds a value that is not finite.
  AKG_DEV bool odd() const {
    typedef u16 u16x2 __attribute__((ext_vector_type(2)));
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, held[i][e] & 0x7fff7fffu));
    }
    return most[0] >= kInfinity || most[1] >= kInfinity;
  }
  // Zeros in place of such values; the first row of each channel that has one (`row0`: of the tile's first), if it comes before what
  // `spoilt` has.
  AKG_DEV void clean(int *spoilt, int row0, int tid) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int c = tid + i * THREADS, row = row0 + c / kPerRow, at = c % kPerRow * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u32 bits = 0x7fffu << 16 * (e & 1);
        if (((held[i][e / 2] & bits) >> 16 * (e & 1)) >= kInfinity) {
          __hip_atomic_fetch_min(spoilt + at + e, row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          held[i][e / 2] &= ~bits;
        }
      }
    }
  }
  AKG_DEV void store(u8 *tile, int tid) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int c = tid + i * THREADS;
      if (!kWhole && c >= kChunks) continue;
      u8 *to = tile + (kEven ? chunk_at<W>(tid / kPerRow, tid % kPerRow) + i * (THREADS / kPerRow) * pitch(W) : chunk_at<W>(c / kPerRow, c % kPerRow));
      if constexpr (PARTS == 1) {
        *reinterpret_cast<u32x4 *>(to) = held[i];
      } else {   // float16
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = attn::F16::low(held[i][e]);
          x[2 * e + 1] = attn::F16::high(held[i][e]);
        }
        u32x4 parts[2];
        split<2>(x, parts);
        *reinterpret_cast<u32x4 *>(to) = parts[0];
        *reinterpret_cast<u32x4 *>(to + kTileBytes) = parts[1];
      }
    }
  }
};

// What the emitted kernel states about a walk: the operands' type, channels of a and b (D) and of c and the result (E), 32-token
// tiles of a chunk (CT), wavefronts that hold the state (NW, 32 channels of c each, times HALVES of its rows), wavefronts that fetch
// and multiply (HELPERS, two or four), whether LDS holds one chunk's tiles only (TIGHT), whether what is added to the state goes in
// three parts instead of two (REST), heads of the states (H) and of each operand, whether it runs backward, whether states given and
// left are the transposed ones ([E][D] in memory).
enum class Result { None, Storage, Float };
template <typename T_, int D_, int E_, int CT_, int NW_, int HALVES_, int HELPERS_, bool TIGHT_, bool REST_, int H_, int HA_, int HB_, int HC_,
          bool HEADS_FIRST_, bool BACK_, bool TURNED_, Result RESULT_>
struct Config {
  typedef T_ T;   // attn::BF16 or attn::F16
  static constexpr int PARTS = T::kNarrowRange ? 2 : 1, D = D_, E = E_, CT = CT_, NW = NW_, HALVES = HALVES_, HELPERS = HELPERS_, H = H_, HA = HA_, HB = HB_, HC = HC_;
  static constexpr bool TIGHT = TIGHT_, REST = REST_, HEADS_FIRST = HEADS_FIRST_, BACK = BACK_, TURNED = TURNED_;
  static constexpr Result RESULT = RESULT_;
  static constexpr int kChunk = 32 * CT, kColumns = 32 * NW, kTiles = (E + kColumns - 1) / kColumns;
};

// Tiles of a few chunks, and masked products as operands. STATES: what a walk over states alone needs.
template <typename C, bool STATES>
struct Lds {
  static constexpr int kPairs = C::CT * (C::CT + 1) / 2;   // 32 x 32 tiles of the masked products
  static constexpr int kA = C::TIGHT ? 1 : 2, kB = C::TIGHT ? 1 : 3;
  u8 b[kB][C::PARTS][C::kChunk * pitch(C::D)], c[kB][C::PARTS][C::kChunk * pitch(C::kColumns)], a[STATES ? 0 : kA][C::PARTS][C::kChunk * pitch(C::D)];
  u32x4 pairs[STATES ? 0 : kA][C::PARTS][kPairs][2][64];
  f32x4 other[STATES || C::HALVES == 1 ? 0 : kA][C::NW][C::CT][4][64];   // a . S of the second half of the rows
  // By every wavefront that fetches: the first token of the segment whose c is not finite, for each channel, and whether there is one.
  int spoilt[STATES ? 0 : C::HELPERS][C::kColumns];
  __attribute__((aligned(16))) int odd[STATES ? 0 : C::HELPERS];
};
constexpr int kNever = 0x7fffffff;

// Where the tokens of one head of a tensor with X heads of W channels of 2 bytes lie.
template <int X, int W, bool HEADS_FIRST, int H>
struct Tokens {
  const char *base;
  long step;
  AKG_DEV Tokens(const void *p, long b, int h, long seq, int size = 2) {
    const long head = h / (H / X);
    step = static_cast<long>(size) * W * (HEADS_FIRST ? 1 : X);
    base = static_cast<const char *>(p) + static_cast<long>(size) * W * (HEADS_FIRST ? (b * X + head) * seq : b * seq * X + head);
  }
};

// A walk's arguments. `starts`: [head][segment][D][E], what every segment adds to a state, left by a walk over states alone, then
// the states in front of them (none where there is one segment).
struct Walk {
  const void *a, *b, *c;
  void *out;
  const float *log_decay, *first;   // [H]; given state (or null)
  float *last;                      // state behind the last token (or null)
  const int *lengths, *slots;       // [batch] or null; slots: which entry of `first` and `last` a sequence has
  float *starts;
  long seq, pool;                   // entries of `first` and `last`
  int segment, segments;            // tokens of a segment (a multiple of the chunk), their number
  float scale;
  bool join;                        // no launch makes the one of the other: a walk adds up what stands in front of its segment
};

AKG_DEV long length_of(const int *lengths, long b, long seq) {
  if (lengths == nullptr) return seq;
  const long n = lengths[b];
  return n < 0 ? 0 : n < seq ? n : seq;
}
// Entry of sequence b in the pool of states, -1: none.
AKG_DEV long entry_of(const int *slots, long b, long pool) {
  if (slots == nullptr) return b;
  const long n = slots[b];
  return n >= 0 && n < pool ? n : -1;
}

// Whether nothing is left of the state given behind the first token, whatever it holds (0 times that may be no number). Backward the
// first token has it already.
template <bool BACK>
AKG_DEV bool forgets(float g, long len) { return !BACK && len > 0 && g == -__builtin_inff(); }

// Tokens of segment s of a sequence of `len`.
AKG_DEV int tokens_of(const Walk &w, long len, int s) {
  const long left = len - static_cast<long>(s) * w.segment;
  return left <= 0 ? 0 : left < w.segment ? static_cast<int>(left) : w.segment;
}

// One segment of one head, 32 NW channels of c. STATES: only what the segment adds to a state.
//
// NW wavefronts hold the state and do what needs it (with HALVES 2 NW, half of the rows each, since a state of 256 leaves a wavefront
// few registers: the second half's a . S reaches the first through LDS). The others fetch into registers, two chunks ahead of what
// they put into LDS (float16 in parts), and compute the masked products. Between two barriers the first have what chunk t adds to
// the state, its masked products with c, and a . S of chunk t + 1; the others the masked products of t + 1, and a, b and c of t + 2
// to put in place of tiles that nothing reads any more. TIGHT: one after the other.
template <typename C, bool STATES>
AKG_DEV void walk(const Walk &w, Lds<C, STATES> &lds, long head, int tile, int seg) {
  constexpr int D = C::D, E = C::E, PARTS = C::PARTS, CT = C::CT, NW = C::NW, kChunk = C::kChunk, kThreads = 64 * C::HELPERS;
  constexpr int kHalves = C::HALVES, kWaves = NW * kHalves, kUnits = whole(D) / 32 / kHalves, kSteps = 2 * CT, kAfter = C::BACK ? 1 : 0;
  constexpr int kTerms = C::REST ? 3 : 2;   // parts of what is added to the state
  constexpr bool TIGHT = C::TIGHT;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), half = lane >> 5;
  const long b = head / C::H;
  const int h = static_cast<int>(head % C::H), e0 = tile * C::kColumns;
  const long len = length_of(w.lengths, b, w.seq);
  const long from = static_cast<long>(seg) * w.segment, upto = from + w.segment < w.seq ? from + w.segment : w.seq, end = upto < len ? upto : len;
  const int chunks = end > from ? static_cast<int>((end - from + kChunk - 1) / kChunk) : 0;
  const float g = w.log_decay[h], g2 = g * kLog2e;
  auto count_of = [&](int t) {
    const long left = end - from - static_cast<long>(t) * kChunk;
    return static_cast<int>(left < kChunk ? (left > 0 ? left : 0) : kChunk);
  };
  // the lowest of the tokens of a chunk, whose last rows they are
  auto lowest_of = [&](int t, int n) {
    const long r0 = from + static_cast<long>(t) * kChunk;
    return C::BACK ? len - r0 - n : r0;
  };
  const Places<D> pd(lane);
  const u8 *mem = reinterpret_cast<const u8 *>(&lds);
  auto place_of = [&](const u8 *tile_) { return static_cast<int>(tile_ - mem); };

  if (wave >= kWaves + C::HELPERS) return;   // (walks of other channels in the same launch have more; who has ended is not waited for)
  if (wave >= kWaves) {
    const int tid = static_cast<int>(threadIdx.x) - 64 * kWaves, helper = wave - kWaves;
    constexpr int kDeep = 2 * kUnits * kHalves;   // of 16 channels
    const Tokens<C::HA, D, C::HEADS_FIRST, C::H> ta(w.a, b, h, w.seq);
    const Tokens<C::HB, D, C::HEADS_FIRST, C::H> tb(w.b, b, h, w.seq);
    const Tokens<C::HC, E, C::HEADS_FIRST, C::H> tc(w.c, b, h, w.seq);
    const int channels = E - e0 < C::kColumns ? E - e0 : C::kColumns;
    typedef Stage<kChunk, D, kThreads, PARTS> StageD;
    typedef Stage<kChunk, C::kColumns, kThreads, PARTS> StageE;
    StageD sa[2], sb[2];
    StageE sc[2];
    // Piece i of all pieces of chunk t's tiles (behind the last chunk nothing is asked of memory).
    constexpr int kPiecesA = STATES ? 0 : StageD::kEach, kPieces = kPiecesA + StageD::kEach + StageE::kEach;
    struct Sources {
      Rows<kChunk, C::BACK> a, b, c;
    };
    auto sources = [&](int t) {
      const int n = count_of(t);
      const long first = lowest_of(t, n);
      return Sources{Rows<kChunk, C::BACK>(ta.base + first * ta.step, ta.step, n, D), Rows<kChunk, C::BACK>(tb.base + first * tb.step, tb.step, n, D),
                     Rows<kChunk, C::BACK>(tc.base + first * tc.step + 2 * e0, tc.step, n, channels)};
    };
    auto fetch_piece = [&](int to, const Sources &from_, int i) {
      if (i < kPiecesA) {
        sa[to].load(from_.a, i, tid);
      } else if (i < kPiecesA + StageD::kEach) {
        sb[to].load(from_.b, i - kPiecesA, tid);
      } else {
        sc[to].load(from_.c, i - kPiecesA - StageD::kEach, tid);
      }
    };
    auto fetch = [&](int to, int t) {
      const Sources from_ = sources(t);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) fetch_piece(to, from_, i);
    };
    // Chunk t's tiles. A value of c that is not finite would spoil rows that do not see it (their weights are 0, and 0 times it is no
    // number): the tile has 0 there, and the rows that do see it, and the state's column, become no numbers behind the walk.
    auto place = [&](int t, int held, int ia, int ib) {
      if constexpr (!STATES) sa[held].store(lds.a[ia][0], tid);
      sb[held].store(lds.b[ib][0], tid);
      if constexpr (!STATES) {   // (behind the others' stores, which then need not wait for c)
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(sc[held].odd()) != 0, 0)) {
          sc[held].clean(lds.spoilt[helper], t * kChunk - (kChunk - count_of(t)), tid);
          if (lane == 0) lds.odd[helper] = 1;
        }
      }
      sc[held].store(lds.c[ib][0], tid);
    };
    // Weights of the masked products (register r: key token 8 (r / 4) + 4 half + r % 4 of its 32, query token lane % 32). Pairs
    // of tiles (query tile, key tile): 0 = (0, 0), 1 = (1, 0), 2 = (1, 1), one to a wavefront, or 0 and 2 to the first of two.
    float mask[16];
    if constexpr (!STATES) {
      const int most = count_of(0);   // (a walk of fewer tokens than a chunk is its first chunk)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int n = (CT == 2 && helper == 1 ? 32 : 0) + (lane & 31) - (8 * (r >> 2) + 4 * half + (r & 3));
        mask[r] = n < 0 || n >= most ? 0.0f : power(g2, n) * w.scale;
      }
    }
    // `load`: what is asked of memory behind every matrix instruction.
    auto pair = [&](int which, int ia, int ib, auto load) {
      const int qt = which > 0 ? 1 : 0, kt = which > 1 ? 1 : 0;
      f32x16 s = {};
      constexpr int kAhead = kDeep * PARTS > 16 ? 2 : 4;   // (as registers allow)
      u32x4 keys[kDeep][PARTS], queries[kDeep][PARTS];
      auto read = [&](int x) {
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          keys[x][p] = pd.row(mem, place_of(lds.b[ib][p]) + 32 * pitch(D) * kt, 0, x);
          queries[x][p] = pd.row(mem, place_of(lds.a[ia][p]) + 32 * pitch(D) * qt, 0, x);
        }
      };
#pragma unroll
      for (int x = 0; x < kAhead && x < kDeep; ++x) read(x);
#pragma unroll
      for (int x = 0; x < kDeep; ++x) {
        __builtin_amdgcn_sched_barrier(0);
        s = product(keys[x], queries[x], s);
        if (x + kAhead < kDeep) read(x + kAhead);
        load(x);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float v[8];
        // (on the diagonal: where the weight is 0 the product does not count, whatever it is)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = qt == kt && mask[8 * x + e] == 0.0f ? 0.0f : s[8 * x + e] * mask[8 * x + e];
        u32x4 parts[PARTS];
        split<PARTS>(v, parts);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) lds.pairs[ia][p][which][x][lane] = parts[p];
      }
    };
    // The masked products of a chunk, and the pieces of chunk t on their way meanwhile.
    auto multiply = [&](int ia, int ib, int to, int t) {
      constexpr int kPairs = CT * (CT + 1) / 2;
      if (STATES || helper >= kPairs) {
        fetch(to, t);
        return;
      }
      const Sources from_ = sources(t);
      pair(helper, ia, ib, [&](int x) {
#pragma unroll
        for (int i = x * kPieces / kDeep; i < (x + 1) * kPieces / kDeep; ++i) fetch_piece(to, from_, i);
      });
      if constexpr (kPairs > C::HELPERS) {
        if (helper == 0) pair(2, ia, ib, [](int) {});
      }
    };
    if (chunks > 0) {
      fetch(0, 0);
      fetch(1, 1);
      if constexpr (!STATES) {
        for (int x = lane; x < C::kColumns; x += 64) lds.spoilt[helper][x] = kNever;
        if (lane == 0) lds.odd[helper] = 0;
      }
      typedef Lds<C, STATES> L;
#pragma unroll
      for (int p = 0; p < PARTS; ++p) {
#pragma unroll
        for (int x = 0; x < L::kB; ++x) clear_padding<kChunk, D, kThreads>(lds.b[x][p], tid);
#pragma unroll
        for (int x = 0; x < L::kA; ++x) {
          if constexpr (!STATES) clear_padding<kChunk, D, kThreads>(lds.a[x][p], tid);
        }
      }
      place(0, 0, 0, 0);
      if constexpr (TIGHT) {
        __syncthreads();
        multiply(0, 0, 0, 2);
      } else {
        fetch(0, 2);
        place(1, 1, 1, 1);
        __syncthreads();
        multiply(0, 0, 1, 3);
      }
      if constexpr (!STATES) __syncthreads();
    }
    // Beside chunk t; `k`: t mod 2.
    int third = 1;   // t + 1 mod 3
    auto beside = [&](auto k, int t) {
      constexpr int K = decltype(k)::value;
      if (t + 1 >= chunks) return;
      if constexpr (TIGHT) {
        __syncthreads();   // (the tiles have been read)
        place(t + 1, 1 - K, 0, 0);
        __syncthreads();
        multiply(0, 0, 1 - K, t + 3);
        if constexpr (!STATES) __syncthreads();
      } else {
        const int then = third + 1 < 3 ? third + 1 : 0;
        place(t + 2, K, K, then);
        multiply(1 - K, third, K, t + 4);
        third = then;
        __syncthreads();
      }
    };
    for (int t = 0; t < chunks; t += 2) {
      beside(attn::IntTag<0>(), t);
      beside(attn::IntTag<1>(), t + 1);
    }
    if constexpr (!STATES && C::RESULT != Result::None) {   // rows behind the length: zeros
      constexpr bool kFloat = C::RESULT == Result::Float;
      constexpr int kSize = kFloat ? 4 : 2, kPieces = C::kColumns * kSize / 16;
      const Tokens<C::H, E, kFloat || C::HEADS_FIRST, C::H> to(w.out, b, h, w.seq, kSize);
      const long none = from > len ? from : len;
      for (long x = tid; x < (upto - none) * kPieces; x += kThreads) {
        const int d = e0 + static_cast<int>(x % kPieces) * (16 / kSize);
        if (d < E) *reinterpret_cast<u32x4 *>(const_cast<char *>(to.base) + (none + x / kPieces) * to.step + kSize * d) = u32x4{0, 0, 0, 0};
      }
    }
    return;
  }

  // Row of unit u in register r: channel 32 u + 16 (r / 8) + 8 half + r % 8.
  // (of unit 0 .. kUnits - 1 of this wavefront's half of the rows)
  const int block = wave % NW, part = wave / NW, unit0 = part * kUnits;
  const int column = e0 + 32 * block + swapped(lane & 31);   // of the state, in this lane
  f32x16 state[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) state[u] = {};
  const long entry = entry_of(w.slots, b, w.pool);
  float *own = w.starts + (w.starts != nullptr ? head * w.segments * (static_cast<long>(D) * E) : 0), *starts = own + seg * (static_cast<long>(D) * E);
  const float *first = w.first != nullptr && entry >= 0 ? w.first + (entry * C::H + h) * (static_cast<long>(D) * E) : nullptr;
  // Walks that join the segments' states take the one given from the last segment's place, which needs none, since the last state may
  // be written over it before another segment's workgroup begins.
  float *copy = own + (w.segments - 1) * (static_cast<long>(D) * E);
  if (!STATES || (w.join && seg == 0)) {
    const bool turned = C::TURNED && (STATES || w.segments == 1);   // (what lies in the workspace never is)
    const float *given = STATES || w.segments == 1 ? first : !w.join ? starts : first != nullptr ? copy : nullptr;
    if (given != nullptr && column < E) {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = 32 * (unit0 + u) + 16 * (r >> 3) + 8 * half + (r & 7);
          if (D == whole(D) || d < D) state[u][r] = given[turned ? static_cast<long>(column) * D + d : static_cast<long>(d) * E + column];
        }
      }
      if (forgets<C::BACK>(g, len)) {   // (behind the loads, which then need not wait for the decay)
#pragma unroll
        for (int u = 0; u < kUnits; ++u) state[u] = {};
      }
#pragma unroll
      for (int u = 0; STATES && u < kUnits; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = 32 * (unit0 + u) + 16 * (r >> 3) + 8 * half + (r & 7);
          if (D == whole(D) || d < D) copy[static_cast<long>(d) * E + column] = state[u][r];
          state[u][r] = 0.0f;
        }
      }
    }
    if (!STATES && w.join && column < E) {
      for (int s = 0; s < seg; ++s) {
        const float *add = starts - static_cast<long>(seg - s) * (D * E);
        const float over = power(g2, tokens_of(w, len, s));
        f32x16 added[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          added[u] = {};
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int d = 32 * (unit0 + u) + 16 * (r >> 3) + 8 * half + (r & 7);
            if (D == whole(D) || d < D) added[u][r] = add[static_cast<long>(d) * E + column];
          }
        }
        // Nothing of nothing, also where the factor is infinite. (A test beside every sum made the loads wait for each other: 4 x 1003
        // tokens of 16/4 heads of 96/80 29 us instead of 25.)
        const float factor = over < __builtin_inff() ? over : 1.0f;
        if (over == __builtin_inff()) {
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
#pragma unroll
            for (int r = 0; r < 16; ++r) state[u][r] = state[u][r] == 0.0f ? 0.0f : state[u][r] * over;
          }
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
#pragma unroll
          for (int r = 0; r < 16; ++r) state[u][r] = __builtin_fmaf(state[u][r], factor, added[u][r]);
        }
      }
    }
  }
  // What a token adds to the state fades with the tokens of its chunk behind it: 16 (kSteps - 1 - s) + 15 - j for token j of step
  // s (the tokens are the last rows of their tile, however few).
  const float grow = C::BACK ? w.scale : 1.0f, show = C::BACK ? 1.0f : w.scale;
  float added[8], steps[kSteps], shown[CT], fade = 0.0f;
  Fade fades;
#pragma unroll
  for (int e = 0; e < 8; ++e) added[e] = power(g2, 15 - (8 * (e >> 2) + 4 * half + (e & 3)) + kAfter) * grow;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int n = 16 * (kSteps - 1 - s);
    steps[s] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, n >= count_of(0) ? 0.0f : power(g2, n))));
  }
  auto weigh = [&](int n) {
    fades.set(g, n);
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const int row = 32 * i + (lane & 31) - (kChunk - n);
      shown[i] = row < 0 ? 0.0f : power(g2, row + 1 - kAfter) * show;
    }
  };
  weigh(count_of(0));
  const Places<C::kColumns> pc(lane);

  // Matrix instructions one by one, each with its share of what stands beside it: operands of later ones read from LDS,
  // values of later ones rounded or weighted. (The barriers keep that order: left to itself the compiler reads an operand in
  // front of its use and waits.)
  f32x16 out[CT];
  constexpr bool kWide = kUnits > 4;   // (few registers to read ahead)
  constexpr int kAll = 2 * kUnits * CT, kAhead = kWide || C::REST ? 3 : 6;
  u32x4 queries[kAll][PARTS];
  auto query = [&](int ia, int y) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) queries[y][p] = pd.row(mem, place_of(lds.a[ia][p]), 32 * (y % CT), 2 * unit0 + y / CT);
  };
  constexpr int kGroup = !kWide && !C::REST ? kUnits : kUnits % 2 == 0 ? 2 : 1, kPasses = PARTS == 1 ? kTerms : 2 * kTerms - 1;   // units of the state at a time
  constexpr int kAllKeys = kSteps * kUnits, kKeysAhead = kWide ? 3 : kGroup;
  u32x4 values[kSteps][PARTS], more[kSteps][kTerms], keys[kAllKeys][PARTS];
  auto key = [&](int ib, int x) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) keys[x][p] = pd.transposed(mem, place_of(lds.b[ib][p]), 16 * (x / kUnits), unit0 + x % kUnits);
  };
  // (pair e of the eight values of step s)
  auto weighted = [&](int s, int e) {
    float lo = BF16::low(values[s][0][e]), hi = BF16::high(values[s][0][e]);
    if constexpr (PARTS == 2) {
      lo += BF16::low(values[s][1][e]);
      hi += BF16::high(values[s][1][e]);
    }
    split_pair<kTerms>(lo * (added[2 * e] * steps[s]), hi * (added[2 * e + 1] * steps[s]), more[s], e);
  };
  // What chunk ib's part of the state begins with.
  auto ready = [&](int ib) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int p = 0; p < PARTS; ++p) values[s][p] = pc.transposed(mem, place_of(lds.c[ib][p]), 16 * s, block);
    }
#pragma unroll
    for (int x = 0; x < kKeysAhead; ++x) key(ib, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) weighted(0, e);
  };
  // a . S with the first kAhead operands read already; the state fades behind its use
  auto through = [&](int ia) {
#pragma unroll
    for (int i = 0; i < CT; ++i) out[i] = {};
    u32x4 parts[2 * kUnits][PARTS];
    // (pair e of the eight rows x)
    auto rounded = [&](int x, int e) {
      const int r = 8 * (x & 1) + 2 * e;
      float lo = state[x >> 1][r], hi = state[x >> 1][r + 1];
      split_pair<PARTS>(lo, hi, parts[x], e);
      if constexpr (PARTS == 1 || !C::REST) {   // (in parts, three of them added, it copied the whole state instead)
        u32 w = parts[x][PARTS - 1][e];
        asm("" : "+v"(w), "+v"(lo), "+v"(hi));   // (rounded before it fades, which then needs no register more)
        parts[x][PARTS - 1][e] = w;
      }
      state[x >> 1][r] = lo * fade;
      state[x >> 1][r + 1] = hi * fade;
    };
#pragma unroll
    for (int e = 0; e < 4; ++e) rounded(0, e);
#pragma unroll
    for (int y = 0; y < kAll; ++y) {
      __builtin_amdgcn_sched_barrier(0);
      const int x = y / CT, i = y % CT;
      out[i] = product(parts[x], queries[y], out[i]);
      if (y + kAhead < kAll) query(ia, y + kAhead);
      if (x + 1 < 2 * kUnits) {
#pragma unroll
        for (int e = i * 4 / CT; e < (i + 1) * 4 / CT; ++e) rounded(x + 1, e);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (kHalves == 2) {
      if (part == 1) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
#pragma unroll
          for (int x = 0; x < 4; ++x) lds.other[ia][block][i][x][lane] = f32x4{out[i][4 * x], out[i][4 * x + 1], out[i][4 * x + 2], out[i][4 * x + 3]};
        }
      }
    }
  };
  if (chunks > 0) {
    __syncthreads();   // (the first tiles are in place)
    if constexpr (!STATES && !TIGHT) {
#pragma unroll
      for (int y = 0; y < kAhead && y < kAll; ++y) query(0, y);
    }
  }
  int third = 0;   // t mod 3
  // What needs the state in front of chunk t, and the tiles that the rest of it begins with.
  auto front = [&](int t) __attribute__((always_inline)) {
    const int n = count_of(t), ia = TIGHT ? 0 : t & 1, ib = TIGHT ? 0 : third;
    if (t > 0 && n != kChunk) weigh(n);
    fade = fades.next();
    if (TIGHT && t > 0) {
      __syncthreads();
      __syncthreads();   // (the chunk's tiles are in place)
    }
    if constexpr (!STATES) {
      if constexpr (TIGHT) {
#pragma unroll
        for (int y = 0; y < kAhead && y < kAll; ++y) query(0, y);
      }
      through(ia);
    }
    ready(ib);
    if (!STATES || (!TIGHT && t > 0)) __syncthreads();
  };
  auto back = [&](int t) __attribute__((always_inline)) {
    const int n = count_of(t), ia = TIGHT ? 0 : t & 1, ib = TIGHT ? 0 : third;
    third = third + 1 < 3 ? third + 1 : 0;
    u32x4 pairs[kSteps][CT][PARTS];
    if constexpr (!STATES) {
      if constexpr (kHalves == 2) {
        if (part == 0) {
#pragma unroll
          for (int i = 0; i < CT; ++i) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const f32x4 v = lds.other[ia][block][i][x][lane];
#pragma unroll
              for (int e = 0; e < 4; ++e) out[i][4 * x + e] += v[e];
            }
          }
        }
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int i = s / 2; i < CT; ++i) {
#pragma unroll
          for (int p = 0; p < PARTS; ++p) pairs[s][i][p] = lds.pairs[ia][p][i == 0 ? 0 : 1 + s / 2][s & 1][lane];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r) state[u][r] *= fade;
      }
    }
    // a result in float32 is one of the walk's own heads, heads first
    constexpr bool kFloat = C::RESULT == Result::Float, kShow = !STATES && C::RESULT != Result::None;
    constexpr int kSize = kFloat ? 4 : 2;
    const Tokens<C::H, E, kFloat || C::HEADS_FIRST, C::H> to(w.out, b, h, w.seq, kSize);
    // (in a scalar register: the compiler would test every store's descriptor for each lane otherwise)
    const int bytes = __builtin_amdgcn_readfirstlane(static_cast<int>(kShow && part == 0 ? records((n - 1) * to.step + static_cast<long>(kSize) * E) : 0));
    const Buffer buf = make_buffer(to.base + lowest_of(t, n) * to.step, bytes);
    // (half x of query tile i: 16 channels of a row in a pair of lanes)
    auto write = [&](int i, int x) {
      const int row = 32 * i + (lane & 31), behind = C::BACK ? kChunk - 1 - row : row - (kChunk - n), d = e0 + 32 * block + 16 * x + 8 * half;
      const u32 off = row >= kChunk - n && d < E ? static_cast<u32>(behind * static_cast<int>(to.step) + kSize * d) : kBeyondEveryBuffer;
      if constexpr (kFloat) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = out[i][8 * x + 4 * y + e];
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), buf, off + (off == kBeyondEveryBuffer ? 0u : 16u * y), 0, 0);
        }
      } else {
        u32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = C::T::pack(out[i][8 * x + 2 * e], out[i][8 * x + 2 * e + 1]);
        __builtin_amdgcn_raw_buffer_store_b128(v, buf, off, 0, 0);
      }
    };
    // What c adds to the state: a few units at a time, first the products with the rests; keys are read ahead, the next tokens
    // weighted. Behind the first units: the masked products with c, then row by row of the result.
    constexpr int kGroups = kAllKeys / kGroup;
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
      const int s = q * kGroup / kUnits, u0 = q * kGroup % kUnits;
#pragma unroll
      for (int pass = 0; pass < kPasses; ++pass) {
#pragma unroll
        for (int v = 0; v < kGroup; ++v) {
          __builtin_amdgcn_sched_barrier(0);
          const int u = u0 + v, x = q * kGroup + v;
          // (parts of the key and of the value, the smallest products first: those below 2^-16, or 2^-24, are left out)
          const int kp = PARTS == 1 ? 0 : pass % 2, mt = PARTS == 1 ? kTerms - 1 - pass : kTerms - 1 - (pass + 1) / 2;
          state[u] = BF16::mma(keys[x][kp], more[s][mt], state[u]);
          if (pass == 0 && x + kKeysAhead < kAllKeys) key(ib, x + kKeysAhead);
          if (u0 == 0 && pass + 1 == kPasses && s + 1 < kSteps) {
#pragma unroll
            for (int e = v * 4 / kGroup; e < (v + 1) * 4 / kGroup; ++e) weighted(s + 1, e);
          }
          if constexpr (!STATES) {
            if (q == 0 && pass == 0) {
#pragma unroll
              for (int r = v * 16 * CT / kGroup; r < (v + 1) * 16 * CT / kGroup; ++r) out[r / 16][r % 16] *= shown[r / 16];
            }
          }
          if constexpr (kShow) {
            if (q > 0 && pass == 0 && v == 0) {
#pragma unroll
              for (int y = (q - 1) * 2 * CT / (kGroups - 1); y < q * 2 * CT / (kGroups - 1); ++y) write(y / 2, y % 2);
            }
          }
          if constexpr (!STATES && !TIGHT) {   // (of the next chunk's a; behind the last one nothing uses them)
            if (q + 1 == kGroups && pass + 1 == kPasses && v == 0) {
#pragma unroll
              for (int y = 0; y < kAhead && y < kAll; ++y) query(1 - ia, y);
            }
          }
        }
      }
      if constexpr (!STATES) {
        if (q == 0) {
#pragma unroll
          for (int z = 0; z < kSteps; ++z) {
#pragma unroll
            for (int i = z / 2; i < CT; ++i) {
              __builtin_amdgcn_sched_barrier(0);
              out[i] = product(values[z], pairs[z][i], out[i]);
            }
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // One body for both where registers hold it (4 x 4096 tokens of 8 heads of 256 231 us with it, 125 without, of 32 of 128 in
  // float16 269, 223; with the last state kept 4 x 2048 of 16/4 heads of 256 111, 115, gradient of 2 x 1021 of 16/4 of 128 45, 47).
  if constexpr (PARTS == 1 && !kWide) {
    for (int t = 0; t < chunks; ++t) {
      front(t);
      back(t);
    }
  } else if (chunks > 0) {
    front(0);
    for (int t = 0;; ++t) {
      back(t);
      if (t + 1 >= chunks) break;
      front(t + 1);
    }
  }

  // Rows from a value of c on that is not finite, and the state's column behind it: no numbers (the tiles had 0 in its place).
  if constexpr (!STATES) {
    int odd = 0;
#pragma unroll
    for (int i = 0; i < C::HELPERS; ++i) odd |= chunks > 0 ? lds.odd[i] : 0;
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(odd) != 0, 0)) {
      auto first_of = [&](int channel) {
        int n = kNever;
#pragma unroll
        for (int i = 0; i < C::HELPERS; ++i) n = n < lds.spoilt[i][channel] ? n : lds.spoilt[i][channel];
        return n;
      };
      if (first_of(column - e0) != kNever) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
#pragma unroll
          for (int r = 0; r < 16; ++r) state[u][r] = __builtin_nanf("");
        }
      }
      if constexpr (C::RESULT != Result::None) {
        constexpr bool kFloat = C::RESULT == Result::Float;
        const Tokens<C::H, E, kFloat || C::HEADS_FIRST, C::H> to(w.out, b, h, w.seq, kFloat ? 4 : 2);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "agent");   // (behind this wavefront's own stores)
        for (int x = 0; part == 0 && x < 32 && e0 + 32 * block + x < E; ++x) {
          for (long i = static_cast<long>(first_of(32 * block + x)) + lane; i < end - from; i += 64) {
            char *at = const_cast<char *>(to.base) + (C::BACK ? len - 1 - from - i : from + i) * to.step;
            if constexpr (kFloat) {
              reinterpret_cast<float *>(at)[e0 + 32 * block + x] = __builtin_nanf("");
            } else {
              reinterpret_cast<u16 *>(at)[e0 + 32 * block + x] = PARTS == 1 ? 0x7fc0 : 0x7e00;
            }
          }
        }
      }
    }
  }

  // a walk over states leaves them in the workspace; else the segment that holds the last token has the last state
  const bool ends = seg == (len > 0 ? static_cast<int>((len - 1) / w.segment) : 0);
  float *to = STATES ? starts : w.last != nullptr && ends && entry >= 0 ? w.last + (entry * C::H + h) * (static_cast<long>(D) * E) : nullptr;
  if (to != nullptr && column < E) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * (unit0 + u) + 16 * (r >> 3) + 8 * half + (r & 7);
        if (D == whole(D) || d < D) to[C::TURNED && !STATES ? static_cast<long>(column) * D + d : static_cast<long>(d) * E + column] = state[u][r];
      }
    }
  }
}

// The states in front of every segment from what the segments add: start[s + 1] = exp(g tokens of s) start[s] + added[s].
// A thread has four adjacent values of one head.
template <typename C>
AKG_DEV void scan(const Walk &w, long heads, long at) {
  constexpr int D = C::D, E = C::E, kEach = D * E / 4;
  const long head = at / kEach;
  if (head >= heads) return;
  const int x = static_cast<int>(at % kEach) * 4, h = static_cast<int>(head % C::H);
  const long b = head / C::H, len = length_of(w.lengths, b, w.seq), entry = entry_of(w.slots, b, w.pool);
  const float g = w.log_decay[h], g2 = g * kLog2e;
  f32x4 start = {};
  if (w.first != nullptr && entry >= 0) {
    const float *given = w.first + (entry * C::H + h) * (static_cast<long>(D) * E);
#pragma unroll
    for (int e = 0; e < 4; ++e) start[e] = given[C::TURNED ? (x % E + e) * D + x / E : x + e];   // (E is a multiple of 4)
    if (forgets<C::BACK>(g, len)) start = {};
  }
  float *to = w.starts + head * w.segments * (static_cast<long>(D) * E) + x;
  constexpr int kAtOnce = 8;   // (asked for together: one behind the other 16 segments of 16 states of 128 x 128 took 16 us)
  for (int s0 = 0; s0 < w.segments; s0 += kAtOnce) {
    f32x4 add[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      add[k] = f32x4{};
      if (s0 + k + 1 < w.segments) __builtin_memcpy(&add[k], to + static_cast<long>(s0 + k) * (D * E), 16);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (s0 + k >= w.segments) break;
      __builtin_memcpy(to + static_cast<long>(s0 + k) * (D * E), &start, 16);
      const float fade = power(g2, tokens_of(w, len, s0 + k));
#pragma unroll
      for (int e = 0; e < 4; ++e) start[e] = __builtin_fmaf(start[e], start[e] == 0.0f ? 0.0f : fade, add[k][e]);   // (nothing of nothing, also where that is infinite)
    }
  }
}

// Gradients of heads that share keys and values: the sum over those heads, in their order. `part`: [batch][H][seq][W] in
// float32; a thread has four channels of one token of one key head.
template <typename T, int W, int H, int HKV, bool HEADS_FIRST>
AKG_DEV void share(const float *part, void *out, long batch, long seq, long at) {
  constexpr int G = H / HKV;
  const long d = at % (W / 4) * 4, token = at / (W / 4) % seq, head = at / (W / 4) / seq;
  if (head >= batch * HKV) return;
  const float *from = part + (head * G * seq + token) * W + d;
  f32x4 sum = {};
#pragma unroll
  for (int k = 0; k < G; ++k) sum += *reinterpret_cast<const f32x4 *>(from + k * seq * W);
  const long b = head / HKV, hkv = head % HKV;
  const u32x2 v = {T::pack(sum[0], sum[1]), T::pack(sum[2], sum[3])};
  *reinterpret_cast<u32x2 *>(static_cast<u16 *>(out) + (HEADS_FIRST ? (head * seq + token) * W : ((b * seq + token) * HKV + hkv) * W) + d) = v;
}

// ---- few tokens: the recurrence itself ----------------------------------------------------------------------------------
// A workgroup has TE channels of v of one head (TE / 4 lanes side by side) and all D channels of k, a thread D / (1024 / TE)
// adjacent ones of those; the state stays in registers over the tokens. Bound by the state, read and written once.
template <typename T, int D, int E, int TE, int H, int HKV, bool HEADS_FIRST, int MOST>
AKG_DEV void tokens(const Walk &w, long head, int tile) {
  constexpr int kLanes = TE / 4, kGroups = 256 / kLanes, kRows = (D + kGroups - 1) / kGroups, kPerWave = 64 / kLanes;
  typedef typename T::dtype::storage S;
  __shared__ float qs[MOST][kGroups * kRows], ks[MOST][kGroups * kRows];
  __shared__ f32x4 parts[MOST][4][kLanes];
  const int tid = static_cast<int>(threadIdx.x), e = tile * TE + tid % kLanes * 4, row0 = tid / kLanes * kRows;
  const long b = head / H;
  const int h = static_cast<int>(head % H);
  const int seq = static_cast<int>(w.seq), len = static_cast<int>(length_of(w.lengths, b, w.seq));
  const long entry = entry_of(w.slots, b, w.pool);
  const bool live = e < E;
  f32x4 state[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) state[r] = {};
  const long at = (entry * H + h) * (static_cast<long>(D) * E) + e;
  if (w.first != nullptr && entry >= 0 && live) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (D % kGroups == 0 || row0 + r < D) __builtin_memcpy(&state[r], w.first + at + static_cast<long>(row0 + r) * E, 16);
    }
  }
  const Tokens<H, D, HEADS_FIRST, H> tq(w.a, b, h, w.seq);
  const Tokens<HKV, D, HEADS_FIRST, H> tk(w.b, b, h, w.seq);
  const Tokens<HKV, E, HEADS_FIRST, H> tv(w.c, b, h, w.seq);
  for (int x = tid; x < len * kGroups * kRows; x += 256) {
    const int t = x / (kGroups * kRows), d = x % (kGroups * kRows);
    qs[t][d] = d < D ? T::dtype::load(reinterpret_cast<const S *>(tq.base + t * tq.step)[d]) * w.scale : 0.0f;
    ks[t][d] = d < D ? T::dtype::load(reinterpret_cast<const S *>(tk.base + t * tk.step)[d]) : 0.0f;
  }
  const float g = w.log_decay[h], fade = power(g * kLog2e, 1);
  const bool forget = forgets<false>(g, len);
  __syncthreads();
  for (int t = 0; t < len; ++t) {
    f32x4 v = {}, out = {};
    if (live) {
      S raw[4];
      __builtin_memcpy(raw, tv.base + t * tv.step + 2 * e, 8);
#pragma unroll
      for (int z = 0; z < 4; ++z) v[z] = T::dtype::load(raw[z]);
    }
    if (forget) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) state[r] = {};
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float k = ks[t][row0 + r], q = qs[t][row0 + r];
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        state[r][z] = __builtin_fmaf(state[r][z], fade, k * v[z]);
        out[z] = __builtin_fmaf(state[r][z], q, out[z]);
      }
    }
#pragma unroll
    for (int step = kLanes; step < 64; step *= 2) {
#pragma unroll
      for (int z = 0; z < 4; ++z) out[z] += __shfl_xor(out[z], step);
    }
    if ((tid & 63) < kLanes) parts[t][tid >> 6][tid & 63] = out;
  }
  if (w.last != nullptr && entry >= 0 && live) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (D % kGroups == 0 || row0 + r < D) __builtin_memcpy(w.last + at + static_cast<long>(row0 + r) * E, &state[r], 16);
    }
  }
  if (w.out == nullptr) return;
  __syncthreads();
  const Tokens<H, E, HEADS_FIRST, H> to(w.out, b, h, w.seq);
  for (int x = tid; x < seq * kLanes; x += 256) {
    const int t = x / kLanes, lane = x % kLanes, d = tile * TE + lane * 4;
    f32x4 sum = {};
    if (t < len) sum = (parts[t][0][lane] + parts[t][1][lane]) + (parts[t][2][lane] + parts[t][3][lane]);
    const u32x2 v = {T::pack(sum[0], sum[1]), T::pack(sum[2], sum[3])};
    if (d < E) __builtin_memcpy(const_cast<char *>(to.base) + t * to.step + 2 * d, &v, 8);
  }
}

}  // namespace linear
}  // namespace akg
