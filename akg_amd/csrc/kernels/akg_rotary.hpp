/**
 * Rotary positions: pairs of channels turned by angles that grow with the position,
 *   y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin,   angle = position * rate of the pair.
 *
 * Angles are counted in turns as 64-bit binary fractions: position * rate modulo 2^64 drops the whole turns exactly, so
 * an angle at position 2^31 is as good as one at 1 (a float32 product is off by hundredths of a turn from a million on). A
 * rate is rounded to 2^-65 turns: an angle is off by 2^-33 turns at position 2^32, by 2^-25 at 2^40, and says nothing near 2^63.
 * What is left of a quarter turn goes through the Taylor series of sine and cosine on [-pi / 4, pi / 4], whose first
 * dropped terms are below 2^-28 there. Bound by memory: a thread turns the pairs of 16-byte accesses of one head (4 x 4096
 * tokens of 32 + 8 heads of 128 channels in bfloat16 take 59 us, 5.7 TB/s; with the angles computed once for two, four
 * and eight heads a thread 2, 6 and 8 % more: the arithmetic hides behind the accesses, the longer chains do not).
 * Tokens with several positions: a table holds the axis of every pair, and pairs of a thread that have one read its position
 * once (three axes, the same tokens, 60.5 us, 5.5 TB/s).
 */
#pragma once

namespace akg {
namespace rotary {

// Sine and cosine of `turns` / 2^64 turns.
AKG_DEV void sine_cosine(u64 turns, float &sine, float &cosine) {
  const u32 quarter = static_cast<u32>((turns + (1ull << 61)) >> 62);
  // distance from the nearest quarter turn, in [-1/8, 1/8] turns
  const int rest = static_cast<int>(static_cast<u32>(turns >> 32) - (quarter << 30));
  const float x = static_cast<float>(rest) * 0x1.921fb6p-30f;   // 2 pi / 2^32
  const float z = x * x;
  float s = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);   // 1/9!, -1/7!
  s = __builtin_fmaf(z, s, 8.3333333e-3f);
  s = __builtin_fmaf(z, s, -1.6666667e-1f);
  s = __builtin_fmaf(x * z, s, x);
  float c = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);   // -1/10!, 1/8!
  c = __builtin_fmaf(z, c, -1.3888889e-3f);
  c = __builtin_fmaf(z, c, 4.1666667e-2f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.0f);
  const bool odd = quarter & 1;
  const float a = odd ? c : s, d = odd ? s : c;
  sine = quarter & 2 ? -a : a;
  cosine = (quarter + 1) & 2 ? -d : d;
}

// One tensor: where its heads lie, in elements. Token t of (batch, position), head h.
template <typename T, int D, int H, bool HEADS_FIRST>
struct Heads {
  AKG_DEV static long at(long b, long s, int h, long seq) {
    return HEADS_FIRST ? ((b * H + h) * seq + s) * D : ((b * seq + s) * H + h) * D;
  }
};

// V consecutive elements as float, in one access per 16 bytes.
template <typename T, int V>
AKG_DEV void get(const typename T::storage *p, float (&x)[V]) {
  load_chunk_unaligned<T, V>(p, x);
}
template <typename T, int V>
AKG_DEV void set(typename T::storage *p, const float (&x)[V]) {
  store_chunk_unaligned<T, V>(p, x);
}

// P pairs of one token in head `h` of a tensor of H heads. `chunk`: which P pairs; behind the pairs come the channels that
// are only copied, 2 P at a time.
template <typename T, int D, int R, int H, int P, bool HEADS_FIRST, bool INTERLEAVED>
AKG_DEV void turn(const typename T::storage *x, typename T::storage *y, long b, long s, long seq, int h, int chunk,
                  const float (&sine)[P], const float (&cosine)[P]) {
  constexpr int kPairs = R / 2 / P;
  const long at = Heads<T, D, H, HEADS_FIRST>::at(b, s, h, seq);
  if (chunk < kPairs) {
    float u[P], v[P];
    if constexpr (INTERLEAVED) {
      float both[2 * P];
      get<T, 2 * P>(x + at + 2 * P * chunk, both);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        u[e] = both[2 * e];
        v[e] = both[2 * e + 1];
      }
    } else {
      get<T, P>(x + at + P * chunk, u);
      get<T, P>(x + at + R / 2 + P * chunk, v);
    }
    float p[P], q[P];
#pragma unroll
    for (int e = 0; e < P; ++e) {
      p[e] = __builtin_fmaf(u[e], cosine[e], -(v[e] * sine[e]));
      q[e] = __builtin_fmaf(v[e], cosine[e], u[e] * sine[e]);
    }
    if constexpr (INTERLEAVED) {
      float both[2 * P];
#pragma unroll
      for (int e = 0; e < P; ++e) {
        both[2 * e] = p[e];
        both[2 * e + 1] = q[e];
      }
      set<T, 2 * P>(y + at + 2 * P * chunk, both);
    } else {
      set<T, P>(y + at + P * chunk, p);
      set<T, P>(y + at + R / 2 + P * chunk, q);
    }
  } else {
    const int d = R + 2 * P * (chunk - kPairs);
    if constexpr ((D - R) % (2 * P) == 0) {
      typename T::storage both[2 * P];
      __builtin_memcpy(both, x + at + d, sizeof(both));
      __builtin_memcpy(y + at + d, both, sizeof(both));
    } else {
      for (int e = d; e < D && e < d + 2 * P; ++e) y[at + e] = x[at + e];
    }
  }
}

}  // namespace rotary
}  // namespace akg
