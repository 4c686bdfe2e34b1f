/**
 * The operators of an attention layer (RotaryEmbedding, Attention, AttentionGrad, CacheAttention, LinearAttention,
 * LinearAttentionGrad): descriptions of one op become an instance of the hand-written kernels in kernels/akg_rotary.hpp,
 * akg_attention.hpp, akg_cache_attention.hpp and akg_linear_attention.hpp.
 * Types, channels, heads, layout and which operands there are go into the source; batch, sequence lengths and the number
 * of blocks are kernel arguments (LoweredKernel::scalarArgs), so calls that differ there share a code object.
 *
 * Times in the comments are of launches one behind another on inputs that no cache holds (copies of 640 MB in turn), with
 * the rule as it is and with the other choice forced; causal and bfloat16 where nothing else is said.
 */
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <sstream>
#include <utility>

#include "HipLowering.h"

namespace akg {
namespace {

using lowering::dtypeTag;

int64_t ceilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Tokens up to which linear attention goes token after token: us that way, in chunks: 16 x 2, 4, 8, 12 of 16/4 heads of 64, float16,
// 4.5, 4.6, 6.2, 7.9 and 6.4; 16 x 2, 4, 8, 16 of 32 heads of 128 12.8, 14.7, 18.2, 24.9 and 21.4, 21.5, 21.7, 22.1.
constexpr int64_t kFewTokens = 8;

class LayerEmitter {
 public:
  // `limit`: bytes of workspace that ranges of an axis may take (0: any number).
  LayerEmitter(const OpGraph &g, const LoweringOptions &options, int64_t limit = 0)
      : g_(g), op_(g.ops[0]), l_(op_.layer), cus_(options.computeUnits), limit_(limit), name_(g.name + (limit > 0 ? "_within" : "")) {}

  LoweredKernel run() {
    for (size_t i = 0; i < g_.outputs.size(); ++i) {
      for (size_t j = i + 1; j < g_.outputs.size(); ++j) {
        if (g_.outputs[i] == g_.outputs[j]) throw LoweringError("op " + op_.name + ": a result is listed twice among the outputs");
      }
    }
    k_.kernelName = name_ + "_kernel";
    k_.family = op_.kind == OpKind::RotaryEmbedding ? KernelFamily::Rotary
                : op_.kind == OpKind::LinearAttention || op_.kind == OpKind::LinearAttentionGrad ? KernelFamily::LinearAttention
                                                                                                 : KernelFamily::Attention;
    switch (op_.kind) {
      case OpKind::RotaryEmbedding: rotary(); break;
      case OpKind::Attention: attention(); break;
      case OpKind::AttentionGrad: attentionGrad(); break;
      case OpKind::LinearAttention: linearAttention(); break;
      case OpKind::LinearAttentionGrad: linearAttentionGrad(); break;
      default: cacheAttention(); break;
    }
    k_.shapeArgs = lowering::buildShapeArgs(g_);
    if (k_.algorithmicBytes == 0) k_.algorithmicBytes = lowering::countAlgorithmicBytes(g_);
    return k_;
  }

 private:
  const OpGraph &g_;
  const OpNode &op_;
  const LayerAttributes &l_;
  const int cus_;
  const int64_t limit_;
  const std::string name_;   // of the kernels
  LoweredKernel k_;

  const TensorValue &in(size_t i) const { return g_.tensor(op_.inputs[i]); }
  std::string inName(size_t i) const { return "in" + std::to_string(in(i).inputIndex); }
  // Argument of result j, or a null pointer where the description does not return it.
  std::string outName(size_t j) const {
    if (j >= op_.outputs.size()) return "nullptr";
    const int index = g_.tensor(op_.outputs[j]).outputIndex;
    return index < 0 ? "nullptr" : "out" + std::to_string(index);
  }
  bool wanted(size_t j) const { return outName(j) != "nullptr"; }

  // (a launch has fewer than 2^32 threads)
  static unsigned checkGrid(int64_t n, int64_t threads) {
    if (n <= 0 || n * threads >= (1LL << 32)) throw LoweringError("more threads than a launch holds");
    return static_cast<unsigned>(n);
  }
  static std::string number(double v) {
    char buf[40];
    std::snprintf(buf, sizeof(buf), "%af", static_cast<double>(static_cast<float>(v)));
    return buf;
  }
  static const char *flag(bool b) { return b ? "true" : "false"; }

  std::string signature(const std::vector<std::string> &scalars, bool workspace) const {
    std::ostringstream o;
    bool first = true;
    auto sep = [&]() -> std::ostringstream & {
      if (!first) o << ", ";
      first = false;
      return o;
    };
    for (size_t i = 0; i < g_.inputs.size(); ++i) sep() << "const " << dtypeTag(g_.tensor(g_.inputs[i]).dtype) << "::storage *in" << i;
    for (size_t i = 0; i < g_.outputs.size(); ++i) sep() << dtypeTag(g_.tensor(g_.outputs[i]).dtype) << "::storage *out" << i;
    for (const std::string &s : scalars) sep() << "long " << s;
    if (workspace) sep() << "float *akg_ws";
    return o.str();
  }
  std::string head(const char *header) const {
    return "// Generated by the akg HIP lowering for gfx950. Op description: " + g_.name + "\n// family: " + kernelFamilyName(k_.family) + ", op: " + op_.name +
           "\n#include \"akg_rt.hpp\"\n" + header + "\n";
  }
  // `wavesPerSimd`: how many the registers have to leave room for (0: the compiler's choice).
  static std::string kernel(const std::string &name, int threads, const std::string &args, const std::string &body, int wavesPerSimd = 0) {
    return "extern \"C\" __global__ __launch_bounds__(" + std::to_string(threads) + (wavesPerSimd ? ", " + std::to_string(wavesPerSimd) : "") + ") void " + name +
           "(" + args + ") {\n" + body + "}\n\n";
  }
  const char *trait() const { return in(0).dtype == DType::BF16 ? "akg::attn::BF16" : "akg::attn::F16"; }

  // ---- RotaryEmbedding ------------------------------------------------------------------------------------------------
  // Which axis every pair turns by, and the how many-th pair of that axis it is.
  std::vector<std::pair<int64_t, int64_t>> axes() const {
    std::vector<std::pair<int64_t, int64_t>> out;
    if (l_.sections.empty()) {
      for (int64_t i = 0; i < l_.rotaryDims / 2; ++i) out.push_back({0, i});
      return out;
    }
    std::vector<int64_t> used(l_.sections.size(), 0);
    size_t a = 0;
    for (int64_t i = 0; i < l_.rotaryDims / 2; ++i) {
      if (l_.axisCycle && i > 0) a = (a + 1) % used.size();
      while (used[a] == l_.sections[a]) a = (a + 1) % used.size();   // (the sections add up to the pairs)
      out.push_back({static_cast<int64_t>(a), used[a]++});
    }
    return out;
  }
  // Turns per position of every pair, as fractions of 2^64.
  std::vector<uint64_t> rates() const {
    std::vector<uint64_t> out;
    const long double twoPi = 6.283185307179586476925286766559005768L;
    for (const std::pair<int64_t, int64_t> &p : axes()) {
      const bool own = l_.axisOwnRates;
      const long double i = static_cast<long double>(own ? p.second : static_cast<int64_t>(out.size()));
      const long double dims = static_cast<long double>(own ? 2 * l_.sections[static_cast<size_t>(p.first)] : l_.rotaryDims);
      long double w = std::pow(static_cast<long double>(l_.base), -2.0L * i / dims);
      if (l_.scaling == LayerAttributes::Scaling::Linear) {
        w /= static_cast<long double>(l_.factor);
      } else if (l_.scaling == LayerAttributes::Scaling::Wavelength) {
        // turns over the original length: at least `high`: as they are; at most `low`: divided; between: both, linearly
        const long double turns = static_cast<long double>(l_.originalLength) * w / twoPi;
        long double share = (turns - static_cast<long double>(l_.low)) / static_cast<long double>(l_.high - l_.low);
        share = std::min(1.0L, std::max(0.0L, share));
        w = (1.0L - share) * w / static_cast<long double>(l_.factor) + share * w;
      }
      out.push_back(static_cast<uint64_t>(std::floor(w / twoPi * 18446744073709551616.0L + 0.5L)));   // (w <= 1: below 2^62)
    }
    return out;
  }

  void rotary() {
    const size_t tensors = op_.inputs.size() - 1;
    const TensorValue &x = in(0), &positions = in(tensors);
    const size_t seqDim = l_.headsFirst ? 2 : 1, headDim = l_.headsFirst ? 1 : 2;
    const int64_t batch = x.shape[0], seq = x.shape[seqDim], dim = x.shape[3], r = l_.rotaryDims;
    if (batch * seq >= (1LL << 31)) throw LoweringError("op " + op_.name + ": more than 2^31 tokens");
    // pairs of a thread: as many as make 16-byte accesses, fewer where the pairs or the copied channels do not divide
    int64_t pairs = x.dtype == DType::F32 ? 4 : 8;
    while (pairs > 1 && ((r / 2) % pairs != 0 || (dim - r) % (2 * pairs) != 0)) pairs /= 2;
    const int64_t chunks = r / 2 / pairs + ceilDiv(dim - r, 2 * pairs);
    std::vector<int64_t> heads;
    int64_t all = 0;
    for (size_t t = 0; t < tensors; ++t) {
      heads.push_back(wanted(t) ? in(t).shape[headDim] : 0);
      all += heads.back();
    }
    const std::vector<uint64_t> rate = rates();
    std::ostringstream o;
    o << head("#include \"akg_rotary.hpp\"\n");
    o << "__device__ const akg::u64 akg_rates[" << rate.size() << "] = {";
    for (size_t i = 0; i < rate.size(); ++i) o << (i ? ", " : "") << rate[i] << "ull";
    o << "};\n\n";
    // Axes: that of every pair, unless the pairs of a thread all have one (their first pair's).
    const std::vector<std::pair<int64_t, int64_t>> axis = axes();
    const bool several = !l_.sections.empty();
    bool mixed = false;
    for (size_t i = 0; several && i < axis.size(); ++i) mixed = mixed || axis[i].first != axis[i / static_cast<size_t>(pairs) * static_cast<size_t>(pairs)].first;
    if (several) {
      o << "__device__ const akg::u8 akg_axes[" << axis.size() << "] = {";
      for (size_t i = 0; i < axis.size(); ++i) o << (i ? ", " : "") << axis[i].first;
      o << "};\n\n";
    }
    std::ostringstream b;
    const size_t positionRank = positions.shape.size() - (several ? 1 : 0);
    const bool perBatch = positionRank == 2 && positions.shape[positions.shape.size() - 2] == batch;
    b << "  constexpr int P = " << pairs << ", CHUNKS = " << chunks << ", HEADS = " << all << ";\n"
      << "  const long at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;\n"
      << "  const long token = at / (CHUNKS * HEADS);\n  if (token >= akg_batch * akg_seq) return;\n"
      << "  const int rest = static_cast<int>(at % (CHUNKS * HEADS)), chunk = rest % CHUNKS, head = rest / CHUNKS;\n"
      << "  const long b = token / akg_seq, s = token % akg_seq;\n"
      << "  float sine[P], cosine[P];\n";
    const std::string stride = perBatch ? "akg_batch * akg_seq" : "akg_seq", place = perBatch ? "token" : "s";
    auto position = [&](const std::string &axisOf) {
      return "const akg::u64 position = static_cast<akg::u64>(static_cast<long long>(" + inName(tensors) + "[" + (several ? axisOf + " * (" + stride + ") + " : "") + place + "]));\n";
    };
    const std::string last = std::to_string(r / 2 - 1);
    if (!mixed) b << "  " << position("static_cast<long>(akg_axes[P * chunk < " + last + " ? P * chunk : " + last + "])");
    b << "#pragma unroll\n  for (int e = 0; e < P; ++e) {\n"
      << "    const int pair = P * chunk + e;\n";
    if (mixed) b << "    " << position("static_cast<long>(akg_axes[pair < " + last + " ? pair : " + last + "])");
    b << "    akg::rotary::sine_cosine(position * akg_rates[pair < " << r / 2 << " ? pair : 0], sine[e], cosine[e]);\n"
      << "    sine[e] *= " << number(l_.inverse ? -l_.magnitude : l_.magnitude) << ";\n    cosine[e] *= " << number(l_.magnitude) << ";\n  }\n";
    int64_t before = 0;
    for (size_t t = 0; t < tensors; ++t) {
      if (heads[t] == 0) continue;
      b << "  " << (before ? "else " : "") << "if (head < " << before + heads[t] << ") akg::rotary::turn<" << dtypeTag(x.dtype) << ", " << dim << ", " << r
        << ", " << heads[t] << ", P, " << flag(l_.headsFirst) << ", " << flag(l_.interleaved) << ">(" << inName(t) << ", " << outName(t)
        << ", b, s, akg_seq, head - " << before << ", chunk, sine, cosine);\n";
      before += heads[t];
    }
    o << kernel(k_.kernelName, 256, signature({"akg_batch", "akg_seq"}, false), b.str());
    k_.source = o.str();
    k_.scalarArgs = {batch, seq};
    k_.grid[0] = checkGrid(ceilDiv(batch * seq * chunks * all, 256), 256);
    k_.block[0] = 256;
    k_.scheduleNote = "pairs per thread " + std::to_string(pairs);
  }

  // ---- Attention and its gradient -------------------------------------------------------------------------------------
  struct Sizes {
    int64_t batch, sq, sk, heads, kvHeads, dk, dv, group, rows, keyHeads;
  };
  Sizes sizes(const TensorValue &q, const TensorValue &k, const TensorValue &v) const {
    const size_t seqDim = l_.headsFirst ? 2 : 1, headDim = l_.headsFirst ? 1 : 2;
    Sizes s;
    s.batch = q.shape[0];
    s.sq = q.shape[seqDim];
    s.sk = k.shape[seqDim];
    s.heads = q.shape[headDim];
    s.kvHeads = k.shape[headDim];
    s.dk = q.shape[3];
    s.dv = v.shape[3];
    s.group = s.heads / s.kvHeads;
    s.rows = s.sq * s.group;
    s.keyHeads = s.batch * s.kvHeads;
    if (s.dk % 8 != 0 || s.dv % 8 != 0 || s.dk > 256 || s.dv > 256) {
      throw LoweringError("op " + op_.name + ": the channels of a head must be a multiple of 8 up to 256");
    }
    // row numbers, key numbers and their sums are 32-bit values, and so are byte offsets between the heads that share a tile of rows
    if (s.rows >= (1LL << 31) - 512 || s.sq + s.sk >= (1LL << 31) - 8192) throw LoweringError("op " + op_.name + ": more than 2^31 rows");
    const int64_t widest = 2 * std::max(s.dk, s.dv);
    if ((l_.headsFirst ? s.group * s.sq * widest : 64 * s.heads * widest) >= (1LL << 31) - 65536 || 64 * s.kvHeads * widest >= (1LL << 31) - 65536) {
      throw LoweringError("op " + op_.name + ": the rows of a tile lie more than 2 GiB apart");
    }
    return s;
  }
  std::string config(const Sizes &s, size_t maskAt) const {
    std::ostringstream o;
    int kind = 0;
    bool mb = false, mh = false, mq = false;
    if (l_.hasMask) {
      const TensorValue &m = in(maskAt);
      kind = m.dtype == DType::Bool ? 1 : m.dtype == DType::F16 ? 2 : m.dtype == DType::BF16 ? 3 : 4;
      mb = m.shape[0] > 1;
      mh = m.shape[1] > 1;
      mq = m.shape[2] > 1;
    }
    o << "typedef akg::attn::Config<" << trait() << ", " << s.dk << ", " << s.dv << ", " << s.kvHeads << ", " << s.group << ", " << flag(l_.headsFirst) << ", "
      << flag(l_.causal) << ", " << kind << ", " << flag(mb) << ", " << flag(mh) << ", " << flag(mq) << "> akg_C;\n\n";
    return o.str();
  }
  // Mask and lengths as arguments of the kernels' functions.
  std::string optionals(size_t at) const {
    std::string s;
    s += l_.hasMask ? inName(at++) : "nullptr";
    s += ", " + (l_.hasQueryLengths ? inName(at++) : std::string("nullptr"));
    s += ", " + (l_.hasKeyLengths ? inName(at++) : std::string("nullptr"));
    return s;
  }
  // Pairs of query and key that see each other where every sequence has its full length.
  static int64_t pairs(const Sizes &s, bool causal) {
    if (!causal) return s.sq * s.sk;
    const int64_t first = s.sk - s.sq + 1, low = std::max<int64_t>(0, 1 - first), n = std::max<int64_t>(0, s.sq - low);
    return n * (first + low) + n * (n - 1) / 2;
  }
  // Workspace of ranges that several workgroups share (attn::Ranges): `groups` counters, `rows` rows over all ranges.
  static int64_t bytesOfRanges(int64_t groups, int64_t rows, int64_t dv) { return ceilDiv(groups * 4, 256) * 256 + rows * (ceilDiv(dv, 32) * 128 + 8); }
  // As many of `splits` ranges as the limit holds.
  int64_t rangesWithin(int64_t splits, int64_t groups, int64_t rows, int64_t dv) const {
    while (limit_ > 0 && splits > 1 && bytesOfRanges(groups, splits * rows, dv) > limit_) --splits;
    return splits;
  }
  static uint64_t rangesBytes(int64_t groups, int64_t rows, int64_t dv) {
    const int64_t bytes = bytesOfRanges(groups, rows, dv);
    if (bytes >= (1LL << 31)) throw LoweringError("the ranges' results take more than 2 GiB");
    return static_cast<uint64_t>(bytes);
  }
  // The kernel `body` whose workgroups (`groups` of `groupRows` rows, times `splits`) share the keys' axis, and what joins
  // their results: the last workgroup of a group, which saves a launch (attention of one query of 8 x 32/8 heads of 128 over 512
  // keys 12.7 instead of 18.3 us), or, where that one would read more than 16 KiB alone, a launch of its own (2 x 16 queries
  // over 8192 keys, 1 MiB a group: 29 instead of 87 us; 4 x 4 over 4096, 128 KiB: 23 instead of 29).
  static constexpr int64_t kJoinInside = 16 << 10;
  static bool joinsInside(int64_t groupRows, int64_t splits, int64_t dv) { return 4 * groupRows * splits * dv <= kJoinInside; }
  void ranges(std::ostringstream &o, const std::string &args, const std::string &body, int threads, int hint, const std::string &joinExtents, const std::string &outs,
              int64_t groups, int64_t groupRows, int64_t splits, int64_t keyHeads, int64_t rows, int64_t dv) {
    k_.workspaceBytes = rangesBytes(groups, splits * keyHeads * rows, dv);
    if (joinsInside(std::min(groupRows, rows), splits, dv)) {
      o << kernel(k_.kernelName, threads, args, body, hint);
      k_.grid[0] = checkGrid(groups * splits, threads);
      k_.block[0] = static_cast<unsigned>(threads);
      return;
    }
    KernelPhase first;
    first.kernelName = name_ + "_ranges";
    first.grid[0] = checkGrid(groups * splits, threads);
    first.block[0] = static_cast<unsigned>(threads);
    k_.earlierPhases.push_back(first);
    const int64_t joinRows = std::max<int64_t>(1, 256 / dv);
    o << kernel(first.kernelName, threads, args, body, hint)
      << kernel(k_.kernelName, 256, args, "  akg::attn::join_rows<akg_C, " + std::to_string(joinRows) + ", " + std::to_string(groupRows) + ">(akg_ws, " + outs + ", " +
                joinExtents + ", static_cast<int>(akg_splits));\n");
    k_.grid[0] = checkGrid(keyHeads * ceilDiv(rows, joinRows), 256);
    k_.block[0] = 256;
  }
  // Wavefronts of a workgroup that gives 32 rows to each (a tile is fetched once for all of them), two at least: the second
  // one fetches even where it has no rows (one query of 8 sequences over 8192 keys with one wavefront 56 us, with two 51).
  // Causal: as many as leave a workgroup for every CU, since rows differ in their keys and many small workgroups even that out
  // (2 x 4096 x 32/8 heads of 128 with eight 313 us, four 328; 1 x 1024 x 16 of 128 with eight, four, two 41, 37, 30).
  // Else the number that puts the fewest on the busiest SIMD: of equals the largest, or the smallest where that is one, which
  // spreads them over most CUs (gradient of 8 x 5792 x 1 of 128: 184 workgroups of eight 526 us, 368 of four 631; of 4 x 2638 x
  // 8/4 of 40: four 303, eight 318; attention of 3 x 478 x 8 of 40: two 15.0, four 15.1, eight 16.4; none of them causal).
  int waves(const Sizes &s, int most) const {
    int w = most;
    if (l_.causal) {
      while (w > 2 && (s.rows <= 32 * (w / 2) || s.keyHeads * ceilDiv(s.rows, 32 * w) < cus_)) w /= 2;
      return w;
    }
    auto load = [&](int n) { return ceilDiv(ceilDiv(s.keyHeads * ceilDiv(s.rows, 32 * n), cus_) * n, 4); };
    for (int n = most / 2; n >= 2; n /= 2) {
      if (load(n) < load(w) || load(n) == 1) w = n;
    }
    return w;
  }

  void attention() {
    const Sizes s = sizes(in(0), in(1), in(2));
    const int nw = waves(s, std::max(s.dk, s.dv) > 128 ? 4 : 8);
    const int64_t groups = s.keyHeads * ceilDiv(s.rows, 32 * nw);
    // Few rows and a long axis of keys: several workgroups share it, as many as two to a CU, or one of eight
    // wavefronts (8 sequences over 8192 keys: 51 us; one to a CU 61), at least two tiles of 64 each (one query of 8 sequences
    // over 512 keys: 12.7 us; four tiles 15.0, one 13.0). A launch that joins has to be worth it (4 x 439 queries and keys of
    // 8/4 heads of 96, not causal: 16.4 us, in two ranges 27.6; 2 x 5 queries over 759 keys of 32/4 of 64, not causal: 19.8
    // in one, 15.0 in two, 12.0 in five).
    int64_t splits = 1;
    if (groups < cus_) splits = std::max<int64_t>(1, std::min<int64_t>({(nw == 8 ? 1 : 2) * cus_ / groups, s.sk / 128, 64}));
    splits = rangesWithin(splits, groups, s.keyHeads * s.rows, s.dv);
    if (!joinsInside(std::min<int64_t>(32 * nw, s.rows), splits, s.dv) && s.sk - s.sk / splits < 512) splits = 1;
    std::ostringstream o;
    o << head("#include \"akg_attention.hpp\"\n") << config(s, 3);
    const std::string args = signature({"akg_batch", "akg_sq", "akg_sk", "akg_splits"}, splits > 1);
    const std::string extents = "akg::attn::Extents{akg_batch, akg_sq, akg_sk}";
    const std::string outs = outName(0) + ", " + outName(1);
    auto call = [&](bool split) {
      return "  akg::attn::forward<akg_C, " + std::to_string(nw) + ", " + flag(split) + ", " +
             flag(split && joinsInside(std::min<int64_t>(32 * nw, s.rows), splits, s.dv)) + ">(" + inName(0) + ", " + inName(1) + ", " + inName(2) + ", " +
             optionals(3) + ", " + outs + ", " + (split ? "akg_ws" : "nullptr") + ", " + extents + ", " + number(l_.scale) + ", static_cast<int>(akg_splits));\n";
    };
    if (!wanted(0)) throw LoweringError("op " + op_.name + ": its first result must be an output");
    if (splits > 1) {
      ranges(o, args, call(true), 64 * nw, 0, extents, outs, groups, 32 * nw, splits, s.keyHeads, s.rows, s.dv);
    } else {
      o << kernel(k_.kernelName, 64 * nw, args, call(false));
      k_.grid[0] = checkGrid(groups, 64 * nw);
      k_.block[0] = static_cast<unsigned>(64 * nw);
    }
    k_.source = o.str();
    k_.scalarArgs = {s.batch, s.sq, s.sk, splits};
    k_.algorithmicOps = static_cast<uint64_t>(2 * (s.dk + s.dv) * s.batch * s.heads * pairs(s, l_.causal));
    k_.scheduleNote = "32 rows per wavefront, wavefronts " + std::to_string(nw) + ", key ranges " + std::to_string(splits);
  }

  void attentionGrad() {
    const Sizes s = sizes(in(1), in(2), in(3));
    // What nobody asks for is not computed: dk and dv need only the rows' values of the kernel of dq, and one of them alone
    // not the products of the other.
    const bool wantDq = wanted(0), wantKeys = wanted(1) || wanted(2);
    const int which = wanted(1) && wanted(2) ? 0 : wanted(1) ? 1 : 2;
    const int rg = std::max(s.dk, s.dv) > 128 ? 1 : 2;
    // A workgroup of the kernel of dk and dv has 128 keys. Where that leaves CUs idle it shares the rows with others, 512 of
    // them each at least (causal: two to a CU, since the first keys have most rows), or has 64. us of the gradient unshared,
    // shared: 1 x 1024 x 16/4 heads of 128 101, 73; 1 x 4096 x 32/4 887, 508. With 128 keys and 64, float16 in launches of
    // their own: 8 x 200 x 12 heads of 64 33.0, 32.0. A mask beside more than 64 channels leaves the registers of two wavefronts
    // a SIMD too few: 64 keys and one (5 x 1773 x 8/4 heads of 96, float16, with a mask: 311, 294).
    // Above 256 channels, where dk and dv are workgroups of their own, this makes twice as many workgroups: 1 x 1024 x 16/4 heads
    // of 256 150 us, with half as many ranges 164, unshared 370; 1 x 2048 x 32/8 529, 489, 761; 2 x 2048 x 32/8 952, 857
    // unshared; 2 x 1024 x 16/8 of 192, not causal, 244, 325 unshared. (No one count of them is best.)
    const bool crowded = l_.hasMask && ceilDiv(s.dk, 32) + ceilDiv(s.dv, 32) > 4;
    const bool apart = which == 0 && ceilDiv(s.dk, 32) + ceilDiv(s.dv, 32) > 8;   // (dk and dv by workgroups of their own)
    // (64 keys also where 128 rows of keys or values lie too far apart for 32-bit offsets)
    const bool far = !l_.headsFirst && 128 * s.kvHeads * 2 * std::max(s.dk, s.dv) >= (1LL << 31) - 65536;
    const bool few = crowded || far;
    const int64_t whole = s.keyHeads * ceilDiv(s.sk, few ? 64 : 128);
    int64_t splits = wantKeys ? std::max<int64_t>(1, std::min((l_.causal ? 2 : 1) * cus_ / whole, s.rows / 512)) : 1;
    const int64_t sumsBytes = 4 * s.keyHeads * s.sk * 32 * (ceilDiv(s.dk, 32) + ceilDiv(s.dv, 32));   // of a range
    // (rows' values and bounds of at most eight wavefronts a workgroup, as below)
    while (limit_ > 0 && splits > 1 && splits * sumsBytes + 4 * s.keyHeads * (3 * s.rows + 2 * (ceilDiv(s.rows, 32) + 8) + 256) + 256 > limit_) --splits;
    const int nwk = !few && (splits > 1 || whole >= cus_) ? 4 : 2;
    const int64_t groups = s.keyHeads * ceilDiv(s.sk, 32 * nwk);
    // Small problems: what both kernels need of the rows in a launch of its own, then both in one launch, side by side, while
    // neither fills the card (float16: 8 x 200 x 12 heads of 64 22.4 us instead of 32.0, 2 x 512 x 12 of 64 22.5 instead of 35.7;
    // with three workgroups a CU 2 x 2000 x 2001 x 16/4 of 128 with a mask, not causal, takes 518 instead of 471).
    const bool together = wantDq && wantKeys && splits == 1 && nwk * rg == 4 && !apart && 2 * (groups + s.keyHeads * ceilDiv(s.rows, 128)) <= 5 * cus_;
    const bool rowsFirst = together || !wantDq;   // (the first launch leaves the rows' values only)
    const int nwq = rowsFirst ? 4 : waves(s, std::max(s.dk, s.dv) > 128 ? 4 : 8);
    const int64_t tilesQ = ceilDiv(s.rows, 32 * nwq);
    std::ostringstream o;
    o << head("#include \"akg_attention.hpp\"\n") << config(s, 6);
    std::vector<std::string> scalars = {"akg_batch", "akg_sq", "akg_sk"};
    if (splits > 1) scalars.push_back("akg_splits");
    const std::string args = signature(scalars, true);
    const std::string extents = "akg::attn::Extents{akg_batch, akg_sq, akg_sk}", ranges = splits > 1 ? "static_cast<int>(akg_splits)" : "1";
    auto queries = [&](int part, const std::string &block, const std::string &lds) {
      return "  akg::attn::backward_queries<akg_C, " + std::to_string(nwq) + ", " + std::to_string(part) + ">(" + inName(0) + ", " + inName(1) + ", " + inName(2) + ", " +
             inName(3) + ", " + inName(4) + ", " + inName(5) + ", " + optionals(6) + ", " + outName(0) + ", akg_ws, " + extents + ", " + number(l_.scale) + ", " + block + ", " +
             lds + ");\n";
    };
    auto keys = [&](const std::string &block, const std::string &lds) {
      return "  akg::attn::backward_keys<akg_C, " + std::to_string(nwk) + ", " + std::to_string(rg) + ", " + std::to_string(nwq) + ", " + flag(splits > 1) + ", " + flag(apart) + ", " +
             std::to_string(which) + ">(" + inName(0) + ", " + inName(1) + ", " + inName(2) + ", " + inName(3) + ", " + optionals(6) + ", " + outName(1) + ", " + outName(2) + ", akg_ws, " +
             extents + ", " + number(l_.scale) + ", " + ranges + ", " + block + ", " + lds + ");\n";
    };
    auto queriesLds = [&](int part) { return "akg::attn::QueriesLds<akg_C, " + std::to_string(nwq) + ", " + std::to_string(part) + ">"; };
    const std::string keysLds = "akg::attn::KeysLds<akg_C, " + std::to_string(nwk) + ", " + std::to_string(rg) + ">";
    const int64_t rowGroups = s.keyHeads * tilesQ;
    // float16: dq needs the largest value of every key head first, beside the rows' own launch or in one of its own
    const bool bounds = in(0).dtype == DType::F16, values = bounds && wantDq;
    const int64_t slices = bounds ? std::min<int64_t>(ceilDiv(s.sk, 128), 256) : 0;
    auto slicesOfValues = [&](const std::string &block) {
      return "  akg::attn::slice_of_values<akg_C>(" + inName(3) + ", " + (l_.hasKeyLengths ? inName(6 + (l_.hasMask ? 1 : 0) + (l_.hasQueryLengths ? 1 : 0)) : std::string("nullptr")) +
             ", akg_ws, " + extents + ", akg_batch * akg_C::HKV * ((akg_sq * akg_C::G + " + std::to_string(32 * nwq - 1) + ") / " + std::to_string(32 * nwq) + ") * " +
             std::to_string(nwq) + ", " + block + ");\n";
    };
    // The launches in their order; the last one is the kernel proper.
    std::vector<KernelPhase> phases;
    auto launch = [&](const char *suffix, bool last, int64_t grid, int threads, const std::string &body, int wavesPerSimd = 0) {
      KernelPhase p;
      p.kernelName = last ? k_.kernelName : name_ + suffix;
      p.grid[0] = checkGrid(grid, threads);
      p.block[0] = static_cast<unsigned>(threads);
      phases.push_back(p);
      o << kernel(p.kernelName, threads, args, body, wavesPerSimd);
    };
    if (values && !rowsFirst) launch("_values", false, s.keyHeads * slices, 256, slicesOfValues("blockIdx.x"));
    const int part = rowsFirst ? 1 : 0;
    std::string rowsBody = "  __shared__ " + queriesLds(part) + " akg_lds;\n";
    if (values && rowsFirst) {
      rowsBody += "  const long akg_rows = akg_batch * akg_C::HKV * ((akg_sq * akg_C::G + " + std::to_string(32 * nwq - 1) + ") / " + std::to_string(32 * nwq) + ");\n" +
                  "  if (blockIdx.x < akg_rows) {\n" + queries(part, "blockIdx.x", "akg_lds") + "  } else {\n" + slicesOfValues("blockIdx.x - akg_rows") + "  }\n";
    } else {
      rowsBody += queries(part, "blockIdx.x", "akg_lds");
    }
    launch(rowsFirst ? "_rows" : "_queries", !wantKeys, rowGroups + (values && rowsFirst ? s.keyHeads * slices : 0), 64 * nwq, rowsBody);
    // per row delta and its log-sum (in two parts for an added mask); float16: what bounds the gradients of the scores
    // (attn::BackwardSpace)
    const bool added = l_.hasMask && in(6).dtype != DType::Bool;
    k_.workspaceBytes = static_cast<uint64_t>(4 * s.keyHeads * ((added ? 3 : 2) * s.rows + (bounds ? 2 * tilesQ * nwq + slices : 0)));
    if (together) {
      launch("_keys", true, groups + rowGroups, 256,
             "  typedef " + queriesLds(2) + " akg_Q;\n  typedef " + keysLds + " akg_K;\n" +
                 "  __shared__ __attribute__((aligned(16))) akg::u8 akg_lds[sizeof(akg_Q) > sizeof(akg_K) ? sizeof(akg_Q) : sizeof(akg_K)];\n" +
                 "  const long akg_keys = akg_batch * akg_C::HKV * ((akg_sk + " + std::to_string(32 * nwk - 1) + ") / " + std::to_string(32 * nwk) + ");\n" +
                 "  if (blockIdx.x < akg_keys) {\n" + keys("blockIdx.x", "*reinterpret_cast<akg_K *>(akg_lds)") + "  } else {\n" +
                 queries(2, "blockIdx.x - akg_keys", "*reinterpret_cast<akg_Q *>(akg_lds)") + "  }\n");
    } else if (wantKeys) {
      launch("_keys", splits == 1, (apart ? 2 : 1) * groups * splits, 64 * nwk * rg, "  __shared__ " + keysLds + " akg_lds;\n" + keys("blockIdx.x", "akg_lds"),
             std::max(s.dk, s.dv) > 128 || nwk == 2 ? 0 : 2);
    }
    if (splits > 1) {
      const int64_t channels = (wanted(1) ? s.dk : 0) + (wanted(2) ? s.dv : 0);
      launch("_join", true, ceilDiv(s.keyHeads * s.sk * (channels / 4), 256), 256,
             "  akg::attn::backward_join<akg_C, " + std::to_string(nwq) + ", " + std::to_string(which) + ">(akg_ws, " + outName(1) + ", " + outName(2) + ", " + extents + ", " + ranges + ");\n");
      k_.workspaceBytes = (k_.workspaceBytes + 255) / 256 * 256 + static_cast<uint64_t>(splits * sumsBytes);
    }
    std::copy(phases.back().grid, phases.back().grid + 3, k_.grid);
    std::copy(phases.back().block, phases.back().block + 3, k_.block);
    phases.pop_back();
    k_.earlierPhases = phases;
    k_.source = o.str();
    k_.scalarArgs = {s.batch, s.sq, s.sk};
    if (splits > 1) k_.scalarArgs.push_back(splits);
    // scores, dout v (but for dv alone), and a product for each result
    const int64_t channels = (2 + (wantDq ? 2 : 0) + (wanted(1) ? 2 : 0)) * s.dk + ((wantDq || wanted(1) ? 2 : 0) + (wanted(2) ? 2 : 0)) * s.dv;
    k_.algorithmicOps = static_cast<uint64_t>(channels * s.batch * s.heads * pairs(s, l_.causal));
    k_.scheduleNote = "32 rows per wavefront, wavefronts " + std::to_string(nwq) + (wantDq ? " (dq)" : " (rows)");
    if (wantKeys) k_.scheduleNote += ", " + std::to_string(nwk) + (which == 0 ? " (dk, dv)" : which == 1 ? " (dk)" : " (dv)") + ", row ranges " + std::to_string(splits);
  }

  // ---- CacheAttention -------------------------------------------------------------------------------------------------
  void cacheAttention() {
    const TensorValue &q = in(0), &cache = in(1), &table = in(5);
    const int64_t batch = q.shape[0], sq = q.shape[1], heads = q.shape[2], dim = q.shape[3];
    const int64_t blocks = cache.shape[0], kvHeads = cache.shape[1], page = cache.shape[2], perSequence = table.shape[1];
    const int64_t group = heads / kvHeads, rows = sq * group;
    if (dim % 16 != 0 || dim > 256) throw LoweringError("op " + op_.name + ": the channels of a head must be a multiple of 16 up to 256");
    if (page % 16 != 0) throw LoweringError("op " + op_.name + ": the tokens of a block must be a multiple of 16");
    if (rows >= (1LL << 30) || perSequence * page >= (1LL << 30)) throw LoweringError("op " + op_.name + ": more than 2^30 tokens or rows");
    const int64_t units = ceilDiv(dim, 64);
    // Tiles of 16 rows a workgroup: as many as registers of two wavefronts a SIMD hold (16 sequences of 4096 tokens, 4 key heads of
    // 128, 64 rows each: two tiles 42 us, four tiles and one wavefront 62; of 256: one tile 81, two 91).
    const int64_t rt = std::min<int64_t>(ceilDiv(rows, 16), std::max<int64_t>(1, 4 / units));
    const int64_t groups = batch * kvHeads * ceilDiv(rows, 16 * rt);
    // Workgroups that share a sequence: two to a CU, with at least one step of 32 tokens for each of their four wavefronts, and
    // up to eight where each has 1024 tokens or more. us at one, two, four, eight to a CU: 4 queries over 16 x 2000 tokens
    // (16/4 heads of 64 channels) 12.5, 13.4, 15.3, 14.7; one over 32 x 8192 .. 16384 tokens (32/8 of 128) 240, 175, 195, 169.
    // (One to a CU is faster where its ranges can be joined without a second launch, and leaves half of the bandwidth unused
    // where tokens are many.)
    const int64_t tokens = perSequence * page;
    const int64_t splits = rangesWithin(std::max<int64_t>(1, std::min<int64_t>({std::max(ceilDiv(2 * cus_, groups), std::min(ceilDiv(8 * cus_, groups), tokens / 1024)),
                                                                                ceilDiv(tokens, 128), 64})),
                                        groups, batch * kvHeads * rows, dim);
    // Registers for two wavefronts a SIMD: 32 rows over 16 x 4096 tokens, 4 key heads of 128, 29 us instead of 40; one query over 16
    // x 8192, 8 key heads of 192 and 256, 76 and 94 instead of 79 and 126 (with three 158, spilled, and 125). Up to 128 channels
    // one tile leaves room for three as it is (asked for, nothing changes).
    std::ostringstream o;
    o << head("#include \"akg_attention.hpp\"\n#include \"akg_cache_attention.hpp\"\n")
      << "typedef akg::attn::Config<" << trait() << ", " << dim << ", " << dim << ", " << kvHeads << ", " << group
      << ", false, true, 0, false, false, false> akg_C;\n\n";
    const std::string args = signature({"akg_batch", "akg_sq", "akg_blocks", "akg_per_sequence", "akg_splits"}, splits > 1);
    auto call = [&](bool split) {
      std::ostringstream c;
      c << "  akg::attn::over_cache<akg_C, " << page << ", " << rt << ", " << flag(split) << ", " << flag(split && joinsInside(std::min(16 * rt, rows), splits, dim)) << ", "
        << flag(tokens <= 128 * splits) << ">(";
      for (size_t i = 0; i < 7; ++i) c << inName(i) << ", ";
      c << outName(0) << ", " << (split ? "akg_ws" : "nullptr") << ", akg::attn::CacheExtents{akg_batch, akg_sq, akg_blocks, akg_per_sequence}, "
        << number(l_.scale) << ", static_cast<int>(akg_splits));\n";
      return c.str();
    };
    const int hint = 2;
    if (splits > 1) {
      ranges(o, args, call(true), 256, hint, "akg::attn::Extents{akg_batch, akg_sq, 0}", outName(0) + ", nullptr", groups, 16 * rt, splits, batch * kvHeads, rows, dim);
    } else {
      o << kernel(k_.kernelName, 256, args, call(false), hint);
      k_.grid[0] = checkGrid(groups, 256);
      k_.block[0] = 256;
    }
    k_.source = o.str();
    k_.scalarArgs = {batch, sq, blocks, perSequence, splits};
    // (of the pool, at most the blocks that the table names)
    const uint64_t live = static_cast<uint64_t>(std::min(blocks, batch * perSequence));
    k_.algorithmicBytes = 2 * live * static_cast<uint64_t>(kvHeads) * static_cast<uint64_t>(page * dim + 4) + 4 * static_cast<uint64_t>(table.numel() + batch) +
                          2 * 2 * static_cast<uint64_t>(q.numel());
    k_.algorithmicOps = static_cast<uint64_t>(4 * dim * batch * heads * sq * perSequence * page);
    k_.scheduleNote = "row tiles " + std::to_string(rt) + ", workgroups per sequence and key head " + std::to_string(splits);
  }

  // ---- LinearAttention and its gradient -------------------------------------------------------------------------------
  // One walk over the tokens (linear::Config): which operands are a, b and c, and what becomes of its result.
  struct WalkOf {
    std::string a, b, c, out, first, last;
    int64_t d, e, ha, hb, hc;
    bool back, turned;
    const char *result;   // of linear::Result
    // The op has the last state as a result, asked for or not: what a description returns does not change the bits of it.
    bool rest;
    int64_t tiles = 1;
  };
  struct LinearSizes {
    int64_t batch, seq, heads, kvHeads, dk, dv, states;
  };
  LinearSizes linearSizes(const TensorValue &q, const TensorValue &v) const {
    const size_t seqDim = l_.headsFirst ? 2 : 1, headDim = l_.headsFirst ? 1 : 2;
    LinearSizes s;
    s.batch = q.shape[0];
    s.seq = q.shape[seqDim];
    s.heads = q.shape[headDim];
    s.kvHeads = v.shape[headDim];
    s.dk = q.shape[3];
    s.dv = v.shape[3];
    s.states = s.batch * s.heads;
    if (s.dk % 8 != 0 || s.dv % 8 != 0 || s.dk > 256 || s.dv > 256) {
      throw LoweringError("op " + op_.name + ": the channels of a head must be a multiple of 8 up to 256");
    }
    // (byte offsets inside a chunk are 32-bit values; tokens of a segment and their exponents too)
    if (64 * s.heads * 2 * std::max(s.dk, s.dv) >= (1LL << 31) - 65536) throw LoweringError("op " + op_.name + ": the tokens of a chunk lie more than 2 GiB apart");
    if (s.seq >= (1LL << 31) - 8192) throw LoweringError("op " + op_.name + ": more than 2^31 tokens");
    return s;
  }
  std::string walkConfig(const WalkOf &w, const LinearSizes &s, int ct, int64_t nw, int halves, int helpers, bool tight) const {
    std::ostringstream o;
    o << "akg::linear::Config<" << trait() << ", " << w.d << ", " << w.e << ", " << ct << ", " << nw << ", " << (w.d > 128 ? halves : 1) << ", " << helpers
      << ", " << flag(tight) << ", " << flag(w.rest) << ", " << s.heads << ", " << w.ha << ", " << w.hb << ", " << w.hc
      << ", " << flag(l_.headsFirst) << ", " << flag(w.back) << ", " << flag(w.turned) << ", akg::linear::Result::" << w.result << ">";
    return o.str();
  }
  // The launches of walks that belong together, the last of them the kernel proper unless `more` follow: with several
  // segments what each adds to the states, the states in front of each, then the walks themselves. `space`: bytes of the
  // workspace in front of theirs. The workspace's bytes are returned.
  int64_t walks(std::ostringstream &o, std::vector<KernelPhase> &phases, std::vector<WalkOf> &all, const LinearSizes &s, const std::string &args, const std::string &decay,
                const std::string &lengths, const std::string &slots, int64_t space, bool more) {
    int64_t widest = 0, deepest = 0, values = 0;
    for (const WalkOf &w : all) {
      widest = std::max(widest, w.e);
      deepest = std::max(deepest, w.d);
      values += w.d * w.e;
    }
    const int parts = in(0).dtype == DType::F16 ? 2 : 1;
    const int64_t units = ceilDiv(widest, 32);
    // Two wavefronts share the rows of 32 columns of a state where one has too few registers for them: above 128 channels with
    // operands in two parts or terms of the state in three (4 x 2048 tokens of 16/4 heads of 256, the last state kept: 113 us instead
    // of 319; float16 248, 941; without that 4 x 4096 of 8 heads in bfloat16 127 with one, 159 with two, its gradient 237, 337).
    bool rest = false;
    for (const WalkOf &w : all) rest = rest || w.rest;
    const int halves = deepest > 128 && (parts == 2 || rest) ? 2 : 1;
    // How many wavefronts hold the state of a workgroup (32 columns each: fewer make more workgroups, which all fetch a and b and
    // multiply them), and how many segments share the tokens (each but the last adds a pass over b and c in front): what is
    // expected to take least. A chunk of 64 tokens of 128 channels takes 1.5, 1.7 and 2.3 us with one, two and four such wavefronts
    // (one workgroup a CU), with terms of the state in three parts some 20 % more, a walk over states alone about half; memory gives
    // 4.8 TB/s; a launch more takes some 5 us, two and a state to be joined 8. us at 4 x 4096 tokens of 32 heads of 128: one 192, two 128,
    // four 160, four and two segments 157; 2 x 2048: one 52, two 60, four 76, four and four segments 57; 16384 of 16 heads, the last
    // state kept: four and 1, 8, 16, 32 segments 597, 148, 107, 123, two and eight 126; 4 x 4096 of 16 heads of 64: one 77, two and 1,
    // 4, 8 segments 93, 49, 55; 4 x 1003 of 16/4 of 96/80: one 31, three and 1, 4 segments 32, 25; gradient of 2 x 1021 of 16/4 heads
    // of 128: one, two, four 68, 44, 51; of 4 x 4096 of 32 heads: two, four 358, 332.
    // A few segments' states are added up by the walks themselves, without a launch for it (1 x 512 tokens of 12 heads of 64 in float16,
    // eight segments, 11.6 us instead of 14.2, 4 x 1003 of 16/4 of 96/80, four, 24.7 instead of 26.9, 2048 of 16 heads of 128, eight, 29.5
    // instead of 30.8; 8192 of 8 heads of 128, sixteen, 49 instead of 45), where a wavefront has at most 128 of their rows (4 x 4096 of 8
    // heads of 256, four, 182 instead of 131).
    auto joins = [&](int64_t segments) { return segments > 1 && segments <= 8 && deepest <= 128 * halves; };
    struct Schedule {
      double time;
      int64_t nw, segments;
      int ct;
      bool tight;
    } best = {};
    auto tilesOf = [&](int64_t nw) {
      int64_t n = 0;
      for (const WalkOf &w : all) n += ceilDiv(w.e, 32 * nw);
      return n;
    };
    for (int64_t nw = std::min<int64_t>(units, 4 / halves); nw >= 1; --nw) {
      if (nw > 2 && nw != ceilDiv(units, ceilDiv(units, 4))) continue;
      // Tiles of a few chunks (linear::Lds, linear::pitch) where LDS holds them, of chunks of 32 tokens before those of one chunk only.
      auto pitchOf = [](int64_t d) { return d <= 32 ? 64 : d <= 64 ? 128 : d <= 128 ? 256 : 512; };
      auto ldsBytes = [&](int64_t tiles) { return parts * (32 * tiles * (5 * pitchOf(deepest) + 3 * pitchOf(32 * nw)) + 2 * 2048 * (tiles * (tiles + 1) / 2)) + (halves == 2 ? 2 * 4096 * nw * tiles : 0) + 512 * nw + 16; };
      int ct = parts == 2 || ldsBytes(2) > 160 * 1024 ? 1 : 2;
      const bool tight = ldsBytes(ct) > 160 * 1024;
      const int64_t groups = s.states * tilesOf(nw), chunks = ceilDiv(s.seq, 32 * ct);
      const double each = (0.9 + ct * ((rest ? 0.33 : 0.15) + (parts == 2 ? 0.08 : 0.026) * static_cast<double>(nw * ceilDiv(deepest, 32)))) * (tight ? 1.5 : 1.0);
      const double bytes = static_cast<double>(2 * s.states * s.seq) / 4.8e6;   // us for a channel of every token
      for (int64_t segments = 1; segments <= std::max<int64_t>(1, std::min<int64_t>(cus_ / groups, chunks / 2)); ++segments) {
        const double steps = static_cast<double>(ceilDiv(chunks, segments));
        double moved = 0.0, movedStates = 0.0;
        for (const WalkOf &w : all) {
          // (a and b once more for every further workgroup of a head, most of it from the L2)
          const double again = 1.0 + 0.2 * static_cast<double>(ceilDiv(w.e, 32 * nw) - 1);
          moved += bytes * (static_cast<double>(2 * w.d) * again + static_cast<double>(2 * w.e));
          movedStates += bytes * (static_cast<double>(w.d) * again + static_cast<double>(w.e));
        }
        // (what chunks take and what memory takes overlap, not wholly)
        auto both = [](double x, double y) { return std::max(x, y) + 0.25 * std::min(x, y); };
        double time = both(static_cast<double>(ceilDiv(groups * segments, cus_)) * steps * each, moved);
        if (segments > 1) {
          time += both(static_cast<double>(ceilDiv(groups * (segments - 1), cus_)) * steps * each * 0.55, movedStates) + (joins(segments) ? 4.6 + 0.4 * static_cast<double>(segments) : 8.0) +
                  static_cast<double>(8 * s.states * segments * values) / 4.8e6;
        }
        if (best.nw == 0 || time < best.time) best = {time, nw, segments, ct, tight};
      }
    }
    const int64_t nw = best.nw;
    const int ct = best.ct;
    const bool tight = best.tight;
    for (WalkOf &w : all) w.tiles = ceilDiv(w.e, 32 * nw);
    const int64_t groups = s.states * tilesOf(nw);
    int64_t segments = best.segments;
    while (limit_ > 0 && segments > 1 && space + 4 * s.states * segments * values > limit_) --segments;
    const int64_t chunk = 32 * ct, segment = ceilDiv(ceilDiv(s.seq, segments), chunk) * chunk;
    segments = ceilDiv(s.seq, segment);
    // Two wavefronts that fetch instead of four where two workgroups to a CU are then resident (gradient of 8 x 200 tokens of 12 heads
    // of 64, float16: 16.7 us instead of 22.6; 8 x 77 with a workgroup a CU 7.5 instead of 7.2).
    int helpers = nw <= 2 && deepest <= 64 && groups * segments > cus_ ? 2 : 4;
    k_.scalarArgs = {s.batch, s.seq, segment, segments};
    if (l_.hasSlots) k_.scalarArgs.push_back(in(4).shape[0]);
    o << "typedef " << walkConfig(all[0], s, ct, nw, halves, helpers, tight) << " akg_C0;\n";
    for (size_t i = 1; i < all.size(); ++i) o << "typedef " << walkConfig(all[i], s, ct, nw, halves, helpers, tight) << " akg_C" << i << ";\n";
    o << "\n";
    const bool join = joins(segments);
    // (one segment is stated as such: its walks have no workspace, and what would read a null one has to be known as dead)
    const std::string parted = segments > 1 ? "static_cast<int>(akg_segments)" : "1";
    int64_t before = space;
    std::vector<std::string> structs;
    for (const WalkOf &w : all) {
      std::ostringstream b;
      b << "{" << w.a << ", " << w.b << ", " << w.c << ", " << w.out << ", " << decay << ", " << w.first << ", " << w.last << ", " << lengths << ", " << slots << ", ";
      if (segments > 1) b << "akg_ws + (" << space / 4 << "L + " << (before - space) / 4 << "L * akg_batch * akg_segments)";
      else b << "nullptr";
      b << ", akg_seq, " << (l_.hasSlots ? "akg_pool" : "akg_batch") << ", static_cast<int>(akg_segment), " << parted << ", " << number(l_.scale) << ", " << flag(join) << "}";
      structs.push_back(b.str());
      before += 4 * s.heads * w.d * w.e;
    }
    const int threads = static_cast<int>(64 * (nw * halves + helpers));
    int hint = 2;
    // A head's workgroups are neighbours on one XCD, whose L2 they share: the walks of a gradient read the same tensors, those
    // backward in time at the same time.
    int64_t tiles = 0;
    for (const WalkOf &w : all) tiles += w.tiles;
    auto body = [&](bool states) {
      std::ostringstream b;
      b << "  const int akg_parts = " << parted << (states ? " - 1" : "") << ";\n  __shared__ __attribute__((aligned(256))) akg::u8 akg_lds[";
      auto lds = [&](size_t i) { return "akg::linear::Lds<akg_C" + std::to_string(i) + ", " + flag(states) + ">"; };
      std::string size = "sizeof(" + lds(0) + ")";
      for (size_t i = 1; i < all.size(); ++i) {
        const std::string other = "sizeof(" + lds(i) + ")";
        size = "(" + size + " > " + other + " ? " + size + " : " + other + ")";
      }
      b << size << "];\n  const int akg_id = akg::xcd_contiguous_id(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));\n  const long akg_head = akg_id / (akg_parts * " << tiles
        << ");\n  int akg_part = static_cast<int>(akg_id % (akg_parts * " << tiles << ")), akg_tile = akg_part % " << tiles << ";\n  akg_part /= " << tiles << ";\n";
      for (size_t i = 0; i < all.size(); ++i) {
        const std::string n = std::to_string(i);
        b << "  if (akg_tile < akg_C" << n << "::kTiles) {\n    const akg::linear::Walk akg_w = " << structs[i] << ";\n    akg::linear::walk<akg_C" << n << ", " << flag(states)
          << ">(akg_w, *reinterpret_cast<" << lds(i) << " *>(akg_lds), akg_head, akg_tile, akg_part);\n    return;\n  }\n  akg_tile -= akg_C" << n << "::kTiles;\n";
      }
      return b.str();
    };
    auto launch = [&](const std::string &name, int64_t grid, int n, const std::string &text, int wavesPerSimd) {
      KernelPhase p;
      p.kernelName = name;
      p.grid[0] = checkGrid(grid, n);
      p.block[0] = static_cast<unsigned>(n);
      phases.push_back(p);
      o << kernel(name, n, args, text, wavesPerSimd);
    };
    if (segments > 1) {
      launch(name_ + "_states", groups * (segments - 1), threads, body(true), hint);
    }
    if (segments > 1 && !join) {
      std::ostringstream b;
      b << "  long akg_at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;\n  const long akg_heads = akg_batch * " << s.heads << ";\n";
      for (size_t i = 0; i < all.size(); ++i) {
        b << "  if (akg_at < akg_heads * " << all[i].d * all[i].e / 4 << ") {\n    const akg::linear::Walk akg_w = " << structs[i] << ";\n    akg::linear::scan<akg_C" << i
          << ">(akg_w, akg_heads, akg_at);\n    return;\n  }\n  akg_at -= akg_heads * " << all[i].d * all[i].e / 4 << ";\n";
      }
      launch(name_ + "_starts", ceilDiv(s.states * values / 4, 256), 256, b.str(), 0);
    }
    launch(more ? name_ + "_walks" : k_.kernelName, groups * segments, threads, body(false), hint);
    k_.scheduleNote = "tokens of a chunk " + std::to_string(chunk) + ", wavefronts " + std::to_string(nw) + ", segments " + std::to_string(segments);
    return segments > 1 ? space + 4 * s.states * segments * values : space;
  }
  void lastPhase(std::vector<KernelPhase> phases) {
    std::copy(phases.back().grid, phases.back().grid + 3, k_.grid);
    std::copy(phases.back().block, phases.back().block + 3, k_.block);
    phases.pop_back();
    k_.earlierPhases = phases;
  }

  void linearAttention() {
    const LinearSizes s = linearSizes(in(0), in(2));
    size_t next = 4;
    const std::string state = l_.hasState ? inName(next++) : "nullptr", slots = l_.hasSlots ? inName(next++) : "nullptr";
    const std::string lengths = l_.hasLengths ? inName(next++) : "nullptr";
    std::ostringstream o;
    o << head("#include \"akg_attention.hpp\"\n#include \"akg_linear_attention.hpp\"\n");
    k_.algorithmicOps = static_cast<uint64_t>(4 * s.states * s.seq * s.dk * s.dv);
    if (l_.hasSlots) {   // (of the pool, at most an entry for every sequence)
      const int64_t idle = std::max<int64_t>(0, in(4).shape[0] - s.batch) * s.heads * s.dk * s.dv;
      k_.algorithmicBytes = lowering::countAlgorithmicBytes(g_) - static_cast<uint64_t>(4 * idle * (wanted(1) ? 2 : 1));
    }
    if (s.seq <= kFewTokens) {
      // Columns of a workgroup: as many as leave two workgroups for every CU.
      int64_t te = 128;
      while (te > 16 && (te / 2 >= s.dv || s.states * ceilDiv(s.dv, te) < 2 * cus_)) te /= 2;
      const int64_t tiles = ceilDiv(s.dv, te);
      std::vector<std::string> scalars = {"akg_batch", "akg_seq"};
      if (l_.hasSlots) scalars.push_back("akg_pool");
      std::ostringstream b;
      b << "  const akg::linear::Walk akg_w = {" << inName(0) << ", " << inName(1) << ", " << inName(2) << ", " << outName(0) << ", " << inName(3) << ", " << state << ", "
        << outName(1) << ", " << lengths << ", " << slots << ", nullptr, akg_seq, " << (l_.hasSlots ? "akg_pool" : "akg_batch") << ", 0, 1, " << number(l_.scale) << "};\n"
        << "  akg::linear::tokens<" << trait() << ", " << s.dk << ", " << s.dv << ", " << te << ", " << s.heads << ", " << s.kvHeads << ", " << flag(l_.headsFirst) << ", " << kFewTokens
        << ">(akg_w, blockIdx.x / " << tiles << ", static_cast<int>(blockIdx.x % " << tiles << "));\n";
      o << kernel(k_.kernelName, 256, signature(scalars, false), b.str());
      k_.scalarArgs = {s.batch, s.seq};
      if (l_.hasSlots) k_.scalarArgs.push_back(in(4).shape[0]);
      k_.grid[0] = checkGrid(s.states * tiles, 256);
      k_.block[0] = 256;
      k_.scheduleNote = "token after token, columns of a workgroup " + std::to_string(te);
      k_.source = o.str();
      return;
    }
    std::vector<std::string> scalars = {"akg_batch", "akg_seq", "akg_segment", "akg_segments"};
    if (l_.hasSlots) scalars.push_back("akg_pool");
    WalkOf w{inName(0), inName(1), inName(2), outName(0), state, outName(1), s.dk, s.dv, s.heads, s.kvHeads, s.kvHeads, false, false, wanted(0) ? "Storage" : "None", op_.outputs.size() > 1};
    std::vector<WalkOf> all{w};
    std::vector<KernelPhase> phases;
    // (whether there is a workspace is known only behind the schedule: the text is made twice where there is none)
    std::ostringstream text;
    k_.workspaceBytes = static_cast<uint64_t>(walks(text, phases, all, s, signature(scalars, true), inName(3), lengths, slots, 0, false));
    if (k_.workspaceBytes == 0) {
      text.str("");
      phases.clear();
      walks(text, phases, all, s, signature(scalars, false), inName(3), lengths, slots, 0, false);
    }
    o << text.str();
    lastPhase(phases);
    k_.source = o.str();
  }

  void linearAttentionGrad() {
    const LinearSizes s = linearSizes(in(1), in(3));
    size_t next = 5;
    const std::string state = l_.hasState ? inName(next++) : "nullptr", dstate = l_.hasStateGradient ? inName(next++) : "nullptr";
    const std::string lengths = l_.hasLengths ? inName(next++) : "nullptr";
    const std::string dout = inName(0), q = inName(1), k = inName(2), v = inName(3);
    std::ostringstream o;
    o << head("#include \"akg_attention.hpp\"\n#include \"akg_linear_attention.hpp\"\n");
    const int64_t h = s.heads, kv = s.kvHeads, rows = s.states * s.seq;
    const bool shared = h != kv;
    // gradients of shared heads: every head's own in float32 first
    const int64_t dkBytes = shared && wanted(1) ? 4 * rows * s.dk : 0, dvBytes = shared && wanted(2) ? 4 * rows * s.dv : 0;
    const std::string dvAt = wanted(1) ? "akg_batch * akg_seq * " + std::to_string(h * s.dk) + "L" : "0L";
    std::vector<WalkOf> all;
    const char *part = shared ? "Float" : "Storage";
    if (wanted(0)) all.push_back({dout, v, k, outName(0), state, "nullptr", s.dv, s.dk, h, kv, kv, false, true, "Storage", false});
    if (wanted(1)) all.push_back({v, dout, q, shared ? "akg_ws" : outName(1), dstate, "nullptr", s.dv, s.dk, kv, h, h, true, true, part, false});
    if (wanted(2) || wanted(3)) {
      all.push_back({k, q, dout, !wanted(2) ? "nullptr" : shared ? "akg_ws + " + dvAt : outName(2), dstate, outName(3), s.dk, s.dv, kv, h, h, true, false, wanted(2) ? part : "None", l_.hasState});
    }
    if (all.empty()) throw LoweringError("op " + op_.name + ": none of its results is an output");
    const bool more = dkBytes + dvBytes > 0;
    const std::vector<std::string> scalars = {"akg_batch", "akg_seq", "akg_segment", "akg_segments"};
    std::vector<KernelPhase> phases;
    std::ostringstream text;
    k_.workspaceBytes = static_cast<uint64_t>(walks(text, phases, all, s, signature(scalars, true), inName(4), lengths, "nullptr", dkBytes + dvBytes, more));
    if (k_.workspaceBytes == 0) {
      text.str("");
      phases.clear();
      walks(text, phases, all, s, signature(scalars, false), inName(4), lengths, "nullptr", 0, more);
    }
    o << text.str();
    if (more) {
      KernelPhase p;
      p.kernelName = k_.kernelName;
      p.grid[0] = checkGrid(ceilDiv(s.batch * kv * s.seq * ((dkBytes ? s.dk : 0) + (dvBytes ? s.dv : 0)) / 4, 256), 256);
      p.block[0] = 256;
      phases.push_back(p);
      std::ostringstream b;
      b << "  long akg_at = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;\n";
      auto one = [&](int64_t d, const std::string &from, const std::string &to) {
        b << "  if (akg_at < akg_batch * akg_seq * " << kv * d / 4 << "L) {\n    akg::linear::share<" << trait() << ", " << d << ", " << h << ", " << kv << ", " << flag(l_.headsFirst) << ">("
          << from << ", " << to << ", akg_batch, akg_seq, akg_at);\n    return;\n  }\n  akg_at -= akg_batch * akg_seq * " << kv * d / 4 << "L;\n";
      };
      if (dkBytes) one(s.dk, "akg_ws", outName(1));
      if (dvBytes) one(s.dv, "akg_ws + " + dvAt, outName(2));
      o << kernel(p.kernelName, 256, signature(scalars, true), b.str());
    }
    lastPhase(phases);
    k_.source = o.str();
    // (both states, and a product for every result)
    k_.algorithmicOps = static_cast<uint64_t>((wanted(0) ? 4 : 0) + (wanted(1) || wanted(2) || wanted(3) ? 2 : 0) + (wanted(1) ? 2 : 0) + (wanted(2) ? 2 : 0)) *
                        static_cast<uint64_t>(s.states * s.seq * s.dk * s.dv);
  }
};

}  // namespace

LoweredKernel lowerLayerToHip(const OpGraph &graph, const LoweringOptions &options) {
  // (operands that other ops compute lie in memory first: the description is cut there)
  if (graph.ops.size() != 1) throw LoweringError("op " + graph.ops[0].name + ": operators of an attention layer are kernels of their own");
  LoweredKernel k = LayerEmitter(graph, options).run();
  const int64_t fixed = 16 << 20;   // what a launch without allocations has
  if (k.workspaceBytes > static_cast<uint64_t>(fixed)) {
    LoweredKernel within = LayerEmitter(graph, options, fixed).run();
    if (within.workspaceBytes <= static_cast<uint64_t>(fixed)) {
      k.source += "\n" + within.source;
      k.withinPhases = within.earlierPhases;
      KernelPhase last;
      last.kernelName = within.kernelName;
      std::copy(within.grid, within.grid + 3, last.grid);
      std::copy(within.block, within.block + 3, last.block);
      k.withinPhases.push_back(last);
      k.withinScalarArgs = within.scalarArgs;
      k.withinWorkspaceBytes = within.workspaceBytes;
    }
  }
  return k;
}

}  // namespace akg
