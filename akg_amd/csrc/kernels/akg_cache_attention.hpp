/**
 * Attention of a few queries over a cache of keys and values held in 8 bits, in blocks ("pages") of tokens that lie
 * anywhere in a pool, with one float32 scale per block and key head:
 *   k[b, j] = key_scale[p, h] key_cache[p, h, j % PAGE],  p = block_table[b, j / PAGE],  likewise v
 *
 * A pass reads every live block once and is bound by that, so nothing is staged: a wavefront takes 32 tokens at a time,
 * its loads go to registers and are requested a step ahead. The products run on v_mfma_f32_16x16x32_f16 with the rows
 * (the queries of the heads that share a key head) as the columns of the results, which makes the probabilities one
 * MFMA leaves in a lane the operand of the next. An 8-bit number is exact in float16: the byte plus 128 becomes the low
 * byte of 1024 + b (one byte permutation for two numbers), less 1152. Which channel or token a lane holds at a
 * contracted position is free as long as both operands agree:
 *   scores: lane (token l % 16, g = l / 16) reads the 16 channels 64 u + 16 g ... of its token
 *   output: lane (l % 16, g) reads a few adjacent channels of the tokens 4 g .. 4 g + 3 of both blocks of sixteen
 * The scale of a key block multiplies the scores in float32. That of a value block multiplies the probabilities, which
 * are rounded to float16 behind it (2^-11 of each), relative to a power of two that puts the row's heaviest product of both so
 * far between 2^12 and 2^14: those of a long tail keep their digits down to 2^-26 of the heaviest, whatever scales lie on blocks
 * that the row does not attend to. That power is the row's own, found from a second running maximum, of score + exponent of the
 * scale, and the accumulators follow it exactly.
 *
 * 32 sequences of 8192 to 16384 tokens, one query of 32 heads over 8 of 128 channels, take 169 us: 4.8 TB/s of the 5.2 that
 * a copy reaches. Short ones wait for what depends on one another (length, block numbers, blocks, the other wavefronts, the
 * other workgroups): 512 tokens of one sequence take 7.5 us, 4 queries over 16 x 2000 tokens, in two launches, 11.0.
 */
#pragma once

namespace akg {
namespace attn {

typedef f32x4 acc4;
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

AKG_DEV acc4 mma16(u32x4 a, u32x4 b, acc4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(F16::frag, a), __builtin_bit_cast(F16::frag, b), c, 0, 0, 0);
}
// Two numbers of a word whose bytes are 128 + the signed number, as float16.
AKG_DEV u32 numbers(u32 biased) {
  const half2_t x = __builtin_bit_cast(half2_t, biased);
  const half2_t less = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  return __builtin_bit_cast(u32, x + less);
}
// Eight adjacent 8-bit numbers (two words) as an operand.
AKG_DEV u32x4 operand_of_bytes(u32 w0, u32 w1) {
  w0 ^= 0x80808080u;
  w1 ^= 0x80808080u;
  return u32x4{numbers(__builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)), numbers(__builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)),
               numbers(__builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)), numbers(__builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u))};
}
// Byte t of two words as two numbers.
template <int t>
AKG_DEV u32 numbers_of_byte(u32 w0, u32 w1) {
  return numbers(__builtin_amdgcn_perm(w1, w0, 0x0c000c00u | static_cast<u32>(t) | (static_cast<u32>(4 + t) << 16)) | 0x64006400u);
}

AKG_DEV float max_groups(float v) {
  v = __builtin_fmaxf(v, lane_partner<16>(v));
  return __builtin_fmaxf(v, lane_partner<32>(v));
}
AKG_DEV float add_groups(float v) {
  v += lane_partner<16>(v);
  return v + lane_partner<32>(v);
}

struct CacheExtents {
  long batch, sq, pages, perSequence;   // sequences, queries of each, blocks in the pool, blocks of a sequence's table
};

// RT: tiles of 16 rows of a workgroup; `splits` workgroups share the tokens of a sequence (1: the result is written; more:
// Ranges), and the last of them joins them (JOIN). ONCE: every wavefront has a step of its own at most, so which one it is
// need not wait for the length.
template <typename C, int PAGE, int RT, bool SPLIT, bool JOIN, bool ONCE>
AKG_DEV void over_cache(const void *q, const void *kcache, const void *vcache, const float *kscale, const float *vscale,
                        const int *table, const int *lengths, void *out, float *ws, CacheExtents e, float scale, int splits) {
  typedef typename C::T T;
  constexpr int D = C::DK, NU = (D + 63) / 64, G = C::G, HKV = C::HKV, kWaves = 4, kStep = 32;
  constexpr bool kWide = D % 64 == 0;   // the channels of a lane adjacent: 4 NU bytes in one load
  __shared__ __attribute__((aligned(16))) float parts[kWaves][4 * NU][16][16];
  __shared__ float tops[kWaves][16], sums[kWaves][16];
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const long rows = e.sq * G, blocks = (rows + 16 * RT - 1) / (16 * RT);
  long id = blockIdx.x;
  const int split = SPLIT ? static_cast<int>(id % splits) : 0;
  if (SPLIT) id /= splits;
  const long row0 = id % blocks * (16 * RT);
  const long head = id / blocks, b = head / HKV, hkv = head % HKV;
  const long most = e.perSequence * PAGE;
  long length = lengths[b];
  length = length < 0 ? 0 : (length < most ? length : most);

  // tokens of this workgroup, whole steps
  const long lastRow = (row0 + 16 * RT < rows ? row0 + 16 * RT : rows) - 1;
  long end = length - e.sq + lastRow / G + 1;
  if (end > length) end = length;
  long steps = end > 0 ? (end + kStep - 1) / kStep : 0, firstStep = 0;
  if (ONCE) {
    firstStep = static_cast<long>(split) * kWaves;
  } else if (SPLIT) {
    const long each = (steps + splits - 1) / splits;
    firstStep = split * each < steps ? split * each : steps;
    steps = firstStep + each < steps ? firstStep + each : steps;
  }

  // queries as operands: channels 64 u + 16 g + 8 x + 0 .. 7; bfloat16 goes to float16 relative to the row's largest
  u32x4 qs[RT][NU][2];
  float factor[RT];
  int seen[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const long row = row0 + 16 * rt + n;
    const bool exists = row < rows;
    const long i = exists ? row / G : 0, h = hkv * G + (exists ? row % G : 0);
    const char *from = static_cast<const char *>(q) + ((b * e.sq + i) * C::H + h) * (2L * D);
    long s = exists ? length - e.sq + i + 1 : 0;
    seen[rt] = static_cast<int>(s < 0 ? 0 : (s < length ? s : length));
    float largest = 0.0f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int at = 64 * u + 16 * g + 8 * x;
        qs[rt][u][x] = exists && (kWide || at < D) ? *reinterpret_cast<const u32x4 *>(from + 2 * at) : u32x4{0, 0, 0, 0};
        if (!T::kNarrowRange) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            largest = __builtin_fmaxf(largest, __builtin_fabsf(T::low(qs[rt][u][x][w])));
            largest = __builtin_fmaxf(largest, __builtin_fabsf(T::high(qs[rt][u][x][w])));
          }
        }
      }
    }
    factor[rt] = scale * kLog2e;
    if (!T::kNarrowRange) {
      largest = max_groups(largest);
      const int up = largest > 0.0f && largest < __builtin_inff() ? __builtin_amdgcn_frexp_expf(largest) : 0;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const u32 two = qs[rt][u][x][w];
            qs[rt][u][x][w] = F16::pack(__builtin_ldexpf(T::low(two), -up), __builtin_ldexpf(T::high(two), -up));
          }
        }
      }
      factor[rt] = __builtin_ldexpf(factor[rt], up);
    }
  }

  acc4 acc[RT][4 * NU];
  float top[RT], sum[RT];
  float heaviest[RT];    // maximum of score + exponent of the value scale (2^exponent is above the scale, at most twice it)
  int reference[RT];     // accumulators are in units of 2^reference (behind the maximum)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = neg_inf();
    sum[rt] = 0.0f;
    heaviest[rt] = neg_inf();
    reference[rt] = 0;
#pragma unroll
    for (int d = 0; d < 4 * NU; ++d) acc[rt][d] = {};
  }
  int lowest = -250;   // of the references: 2^-120 of the largest scale so far, so that scales over references stay finite

  struct Step {
    u32x4 k[2][NU];
    u32 v[2][4][NU];
    float ks[2], vs[2];
    bool ok[2];
  };
  // Page of the sixteen tokens from 32 step + 16 x on (-1: none, or outside the pool).
  auto page_of = [&](long step, int x) {
    const long j = step * kStep + 16 * x, at = j / PAGE;
    const long p = table[b * e.perSequence + (at < e.perSequence ? at : 0)];   // (asked for before the length is known)
    return step < steps && j < end && p >= 0 && p < e.pages ? p : -1L;
  };
  auto fetch = [&](Step &s, long step, const long (&page)[2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      s.ok[x] = page[x] >= 0;
      const long p = s.ok[x] ? page[x] : 0;
      const long unit = p * HKV + hkv;
      const long at = (unit * PAGE + (step * kStep + 16 * x) % PAGE) * D;
      s.ks[x] = s.ok[x] ? kscale[unit] : 0.0f;
      s.vs[x] = s.ok[x] ? vscale[unit] : 0.0f;
      const char *kp = static_cast<const char *>(kcache) + at + n * D;
      const char *vp = static_cast<const char *>(vcache) + at + 4 * g * D;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int d = 64 * u + 16 * g;
        s.k[x][u] = s.ok[x] && (kWide || d < D) ? *reinterpret_cast<const u32x4 *>(kp + d) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (kWide) {
          if (s.ok[x]) {
            __builtin_memcpy(s.v[x][r], __builtin_assume_aligned(vp + r * D + 4 * NU * n, 4 * NU == 12 ? 4 : 4 * NU), 4 * NU);
          } else {
#pragma unroll
            for (int u = 0; u < NU; ++u) s.v[x][r][u] = 0;
          }
        } else {
#pragma unroll
          for (int u = 0; u < NU; ++u) {
            const int d = 64 * u + 4 * n;
            s.v[x][r][u] = s.ok[x] && d < D ? *reinterpret_cast<const u32 *>(vp + r * D + d) : 0u;
          }
        }
      }
    }
  };

  long step = firstStep + wave;
  Step now, next;
  long page[2] = {page_of(step, 0), page_of(step, 1)};
  if (step < steps) fetch(now, step, page);
  if (!ONCE) {
    page[0] = page_of(step + kWaves, 0);
    page[1] = page_of(step + kWaves, 1);
  }
  for (; step < steps; step += kWaves) {
    if (!ONCE) {
      if (step + kWaves < steps) fetch(next, step + kWaves, page);
      page[0] = page_of(step + 2 * kWaves, 0);
      page[1] = page_of(step + 2 * kWaves, 1);
    }
    // scores of 2 x 16 tokens
    acc4 s[RT][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][x] = {};
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const u32x4 a0 = operand_of_bytes(now.k[x][u][0], now.k[x][u][1]), a1 = operand_of_bytes(now.k[x][u][2], now.k[x][u][3]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          s[rt][x] = mma16(a0, qs[rt][u][0], s[rt][x]);
          s[rt][x] = mma16(a1, qs[rt][u][1], s[rt][x]);
        }
      }
    }
    // exponents of the scales of the values (zero, and what is no number, weighs nothing)
    float exponent[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float size = __builtin_fabsf(now.vs[x]);
      const bool weighs = size > 0.0f && size < __builtin_inff();
      const int e = __builtin_amdgcn_readfirstlane(weighs ? __builtin_amdgcn_frexp_expf(size) : -1000);   // (the same in all lanes)
      exponent[x] = e > -1000 ? static_cast<float>(e) : neg_inf();
      lowest = e - 120 > lowest ? e - 120 : lowest;
    }
    u32x4 p[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float peaks[2] = {neg_inf(), neg_inf()};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float f = factor[rt] * now.ks[x];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const long j = step * kStep + 16 * x + 4 * g + r;
          s[rt][x][r] = now.ok[x] && j < seen[rt] ? s[rt][x][r] * f : neg_inf();
          peaks[x] = __builtin_fmaxf(peaks[x], s[rt][x][r]);
        }
      }
      const float peak = max_groups(__builtin_fmaxf(peaks[0], peaks[1]));
      // (32 tokens of one block have one scale)
      const float heavy = PAGE % kStep == 0 ? peak + exponent[0] : max_groups(__builtin_fmaxf(peaks[0] + exponent[0], peaks[1] + exponent[1]));
      const float m = __builtin_fmaxf(top[rt], peak);
      const float base = m == neg_inf() ? 0.0f : m;
      const float shrink = __builtin_amdgcn_exp2f(top[rt] - base);
      top[rt] = m;
      sum[rt] *= shrink;
      const float before = heaviest[rt];
      heaviest[rt] = __builtin_fmaxf(before, heavy);
      int unit = reference[rt];
      if (heaviest[rt] > neg_inf()) {
        unit = static_cast<int>(__builtin_floorf(__builtin_fmaxf(heaviest[rt] - base - 13.0f, -250.0f)));   // (at most 115)
        unit = unit > lowest ? unit : lowest;
      }
      const float all = __builtin_ldexpf(shrink, before > neg_inf() ? reference[rt] - unit : 0);   // (at most 2)
      reference[rt] = unit;
      float w[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {   // (a block that the row does not see may have any scale: 0 NaN is no number)
        w[x] = step * kStep + 16 * x < seen[rt] ? __builtin_ldexpf(now.vs[x], -unit) : 0.0f;
      }
#pragma unroll
      for (int d = 0; d < 4 * NU; ++d) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[rt][d][r] *= all;
      }
      float e8[8];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = __builtin_amdgcn_exp2f(s[rt][x][r] - base);
          sum[rt] += y;
          e8[4 * x + r] = y * w[x];
        }
      }
#pragma unroll
      for (int z = 0; z < 4; ++z) p[rt][z] = F16::pack(e8[2 * z], e8[2 * z + 1]);
    }
    // output: channel (u, t) of lane n, tokens 4 g .. 4 g + 3 of both sixteens
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      u32 word[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int r = 0; r < 4; ++r) word[x][r] = now.v[x][r][u] ^ 0x80808080u;
      }
      auto column = [&](auto tag) {
        constexpr int t = decltype(tag)::value;
        const u32x4 a = {numbers_of_byte<t>(word[0][0], word[0][1]), numbers_of_byte<t>(word[0][2], word[0][3]),
                         numbers_of_byte<t>(word[1][0], word[1][1]), numbers_of_byte<t>(word[1][2], word[1][3])};
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) acc[rt][4 * u + t] = mma16(a, p[rt], acc[rt][4 * u + t]);
      };
      column(IntTag<0>());
      column(IntTag<1>());
      column(IntTag<2>());
      column(IntTag<3>());
    }
    if (ONCE) break;
    now = next;
  }

  // the four wavefronts joined, one tile of rows at a time; then thread (row, channels) writes
  const Ranges<C> ranges(ws, e.batch * HKV * blocks, e.batch * HKV * rows, splits);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float own = add_groups(sum[rt]);
    if (rt > 0) __syncthreads();
    if (g == 0) {
      tops[wave][n] = top[rt];
      sums[wave][n] = own;
    }
    const float unit = __builtin_ldexpf(1.0f, reference[rt]);
#pragma unroll
    for (int d = 0; d < 4 * NU; ++d) {
#pragma unroll
      for (int r = 0; r < 4; ++r) parts[wave][d][4 * g + r][n] = acc[rt][d][r] * unit;
    }
    __syncthreads();
    const int row16 = tid & 15;
    const long row = row0 + 16 * rt + row16;
    float m = neg_inf(), total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = __builtin_fmaxf(m, tops[w][row16]);
    const float base = m == neg_inf() ? 0.0f : m;
    float weight[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      weight[w] = __builtin_amdgcn_exp2f(tops[w][row16] - base);
      total = __builtin_fmaf(sums[w][row16], weight[w], total);
    }
    if (row < rows) {
      const long i = row / G, h = hkv * G + row % G;
      const long slot = head * rows + row;
      const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
      // 16 channel positions x 4 NU tiles: position m of tile 4 u + t is channel 4 NU m + 4 u + t (64 u + 4 m + t)
      for (int c = tid >> 4; c < 16 * NU; c += 16) {
        const int m16 = c / NU, u = c % NU;
        const int d = kWide ? 4 * NU * m16 + 4 * u : 64 * u + 4 * m16;
        if (!kWide && d >= D) continue;
        float y[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          y[t] = 0.0f;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) y[t] = __builtin_fmaf(parts[w][4 * u + t][m16][row16], weight[w], y[t]);
        }
        if (SPLIT) {
          ws_store_chunk<4>(ranges.ws, ranges.accumulator(split, slot, d), y);
        } else {
          const u32x2 two = {T::pack(y[0] * inverse, y[1] * inverse), T::pack(y[2] * inverse, y[3] * inverse)};
          *reinterpret_cast<u32x2 *>(static_cast<char *>(out) + ((b * e.sq + i) * C::H + h) * (2L * D) + 2 * d) = two;
        }
      }
      if (SPLIT && tid < 16) {
        const float state[2] = {m, total};
        ws_store_chunk<2>(ranges.ws, ranges.state(split, slot), state);
      }
    }
  }
  if (SPLIT) {
    static_assert(sizeof(parts) >= sizeof(Meeting<64 * kWaves>), "the join meets where the wavefronts did");
    auto &meet = reinterpret_cast<Meeting<64 * kWaves> &>(parts);
    if (!JOIN || !last_workgroup(ranges.counters, id, splits, tid, &meet.flag)) return;
    const long count = rows - row0 < 16 * RT ? rows - row0 : 16 * RT;
    join<C, 64 * kWaves>(ranges, meet, b, hkv, row0, head * rows + row0, static_cast<int>(count), out, nullptr, Extents{e.batch, e.sq, 0}, tid);
  }
}

}  // namespace attn
}  // namespace akg
