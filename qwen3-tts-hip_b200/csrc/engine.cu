// Host engine for the B200 Qwen3-TTS token loop, and the C ABI of qtts_b200.h.
//
// Mirrors piedshag/qwen3-tts-hip's HipTtsEngine (src/generation.rs) around
// the sm_100a kernels of kernels.cu:
//   load                 HipTtsEngine::load_with_options   generation.rs:284-315
//   text prep on device  TtsTextPrep::prepare_*            text.rs:348-382,516-603
//   talker prefill       HipTalker::prefill_token*         talker.rs:207-233
//   frame loop           HipTtsEngine::rollout             generation.rs:657-749
//   streams              HipTtsStream / PollingTextStream  generation.rs:876-963,1086-1451
// Every frame (15 CodePredictor groups + talker decode step + token
// selection) is one CUDA graph launch; loop state lives on the device, so a
// whole generation is enqueued without host round trips and the host reads
// the codes once at the end (or once per stream chunk).
#include <fcntl.h>
#include <sys/mman.h>
#include <sys/stat.h>
#include <unistd.h>

#include <algorithm>
#include <cstdlib>
#include <cmath>
#include <cstring>
#include <deque>
#include <map>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>
#include <unordered_map>
#include <vector>

#include "codec.h"
#include "error.h"
#include "gemm_tc.h"
#include "json.h"
#include "kernels.h"
#include "kv.h"
#include "qtts_b200.h"

namespace qtts {

std::string& last_error() {
  thread_local std::string message;
  return message;
}

namespace {

constexpr uint64_t kSeedXor = 0x9e3779b97f4a7c15ull;  // generation.rs:667
constexpr int kNewline = 198;                          // text.rs:15
constexpr int kTalkerPageShift = 5;                    // 32 positions per KV page

// ---------------------------------------------------------------------------
// safetensors (8-byte LE header length, JSON header, raw little-endian data)
// ---------------------------------------------------------------------------
struct TensorRef {
  std::string dtype;
  std::vector<long long> shape;
  const uint8_t* data = nullptr;
  size_t nbytes = 0;
  long long numel() const {
    long long n = 1;
    for (long long s : shape) n *= s;
    return n;
  }
};

class SafeTensors {
 public:
  explicit SafeTensors(const std::string& path) {
    fd_ = ::open(path.c_str(), O_RDONLY);
    if (fd_ < 0) fail(QTTS_ERR_IO, "failed to open " + path);
    struct stat sb;
    if (fstat(fd_, &sb) != 0 || sb.st_size < 8) fail(QTTS_ERR_IO, "bad safetensors file " + path);
    size_ = (size_t)sb.st_size;
    map_ = mmap(nullptr, size_, PROT_READ, MAP_PRIVATE, fd_, 0);
    if (map_ == MAP_FAILED) fail(QTTS_ERR_IO, "mmap failed for " + path);
    const uint8_t* p = static_cast<const uint8_t*>(map_);
    uint64_t hlen = 0;
    std::memcpy(&hlen, p, 8);
    if (8 + hlen > size_) fail(QTTS_ERR_IO, "truncated safetensors header in " + path);
    try {
      header_ = Json::parse(reinterpret_cast<const char*>(p + 8), hlen);
    } catch (const std::exception& e) {
      fail(QTTS_ERR_IO, std::string("bad safetensors header: ") + e.what());
    }
    base_ = p + 8 + hlen;
    data_size_ = size_ - 8 - hlen;
  }
  ~SafeTensors() {
    if (map_ && map_ != MAP_FAILED) munmap(map_, size_);
    if (fd_ >= 0) ::close(fd_);
  }
  TensorRef get(const std::string& name) const {
    if (!header_.has(name)) invalid("failed to load " + name + ": tensor not found");
    const Json& m = header_.at(name);
    TensorRef t;
    t.dtype = m.string("dtype");
    for (const Json& s : m.at("shape").arr) t.shape.push_back((long long)s.num);
    const Json& off = m.at("data_offsets");
    const size_t b = (size_t)off.arr.at(0).num, e = (size_t)off.arr.at(1).num;
    if (e < b || e > data_size_) fail(QTTS_ERR_IO, "tensor " + name + " outside file");
    t.data = base_ + b;
    t.nbytes = e - b;
    const size_t esz = t.dtype == "BF16" ? 2 : t.dtype == "F32" ? 4 : 0;
    if (esz == 0) invalid(name + " has dtype " + t.dtype + ", expected F32 or BF16");
    if ((size_t)t.numel() * esz != t.nbytes) fail(QTTS_ERR_IO, "tensor " + name + " size mismatch");
    return t;
  }

 private:
  int fd_ = -1;
  void* map_ = nullptr;
  size_t size_ = 0, data_size_ = 0;
  const uint8_t* base_ = nullptr;
  Json header_;
};

uint16_t f32_to_bf16(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);
  u += 0x7fffu + ((u >> 16) & 1u);
  return (uint16_t)(u >> 16);
}
float bf16_to_f32(uint16_t b) {
  uint32_t u = (uint32_t)b << 16;
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}

// ---------------------------------------------------------------------------
// configuration (src/model/config.rs:47-150)
// ---------------------------------------------------------------------------
struct StackCfg {
  int hidden, intermediate, layers, q_heads, kv_heads, head_dim, vocab, groups;
  float eps, theta;
};

struct ModelCfg {
  StackCfg talker, cp;
  int codec_bos, codec_eos, codec_pad, codec_think, codec_think_bos, codec_think_eos;
  std::map<std::string, int> language_ids, speaker_ids;
  int tts_pad, tts_bos, tts_eos, im_start, assistant;
};

StackCfg stack_cfg(const Json& j) {
  StackCfg c;
  c.hidden = (int)j.integer("hidden_size");
  c.intermediate = (int)j.integer("intermediate_size");
  c.layers = (int)j.integer("num_hidden_layers");
  c.q_heads = (int)j.integer("num_attention_heads");
  c.kv_heads = (int)j.integer("num_key_value_heads");
  c.head_dim = (int)j.integer("head_dim");
  c.vocab = (int)j.integer("vocab_size");
  c.groups = (int)j.integer("num_code_groups");
  c.eps = (float)j.number("rms_norm_eps");
  c.theta = (float)j.number("rope_theta");
  return c;
}

ModelCfg load_config(const std::string& dir) {
  const std::string path = dir + "/config.json";
  FILE* f = std::fopen(path.c_str(), "rb");
  if (!f) invalid("failed to read " + path);
  std::string text;
  char buf[65536];
  size_t n;
  while ((n = std::fread(buf, 1, sizeof buf, f)) > 0) text.append(buf, n);
  std::fclose(f);
  Json raw;
  try {
    raw = Json::parse(text.data(), text.size());
  } catch (const std::exception& e) {
    invalid("failed to parse " + path + ": " + e.what());
  }
  ModelCfg m;
  try {
    const Json& t = raw.at("talker_config");
    m.talker = stack_cfg(t);
    m.cp = stack_cfg(t.at("code_predictor_config"));
    m.codec_bos = (int)t.integer("codec_bos_id");
    m.codec_eos = (int)t.integer("codec_eos_token_id");
    m.codec_pad = (int)t.integer("codec_pad_id");
    m.codec_think = (int)t.integer("codec_think_id");
    m.codec_think_bos = (int)t.integer("codec_think_bos_id");
    m.codec_think_eos = (int)t.integer("codec_think_eos_id");
    for (auto& kv : t.at("codec_language_id").obj) m.language_ids[kv.first] = (int)kv.second.num;
    for (auto& kv : t.at("spk_id").obj) m.speaker_ids[kv.first] = (int)kv.second.num;
    m.tts_pad = (int)raw.integer("tts_pad_token_id");
    m.tts_bos = (int)raw.integer("tts_bos_token_id");
    m.tts_eos = (int)raw.integer("tts_eos_token_id");
    m.im_start = (int)raw.integer("im_start_token_id");
    m.assistant = (int)raw.integer("assistant_token_id");
  } catch (const QttsError&) {
    throw;
  } catch (const std::exception& e) {
    invalid("failed to parse " + path + ": " + e.what());
  }
  return m;
}

// ---------------------------------------------------------------------------
// device memory
// ---------------------------------------------------------------------------
class Arena {
 public:
  ~Arena() {
    for (void* p : ptrs_) cudaFree(p);
  }
  template <typename T>
  T* alloc(size_t count) {
    void* p = nullptr;
    const size_t bytes = std::max<size_t>(count * sizeof(T), 16);
    QCK(cudaMalloc(&p, bytes));
    QCK(cudaMemset(p, 0, bytes));
    // The zeroing runs on the legacy stream, which the engine's non-blocking
    // stream does not wait for: finish it before anything is uploaded into
    // the new buffer on that stream.
    QCK(cudaStreamSynchronize(0));
    ptrs_.push_back(p);
    bytes_ += bytes;
    return static_cast<T*>(p);
  }
  size_t bytes() const { return bytes_; }

 private:
  std::vector<void*> ptrs_;
  size_t bytes_ = 0;
};

struct DevStack {
  StackCfg c;
  int q_out, kv_out, qkv_w;
  std::vector<__nv_bfloat16*> wqkv, wo, wgu, wdown;
  std::vector<float*> in_g, post_g, q_g, k_g;
  float* rope_cos = nullptr;
  float* rope_sin = nullptr;
};

struct StackBufs {
  float *x, *qkv, *q, *attn, *h1, *act;
};

struct SampleKey {
  SampleCfg t, s;
  float penalty;
  int last;
  bool operator<(const SampleKey& o) const { return std::memcmp(this, &o, sizeof *this) < 0; }
};

SampleCfg talker_cfg(const qtts_generate_options& o) {
  return SampleCfg{o.do_sample ? 1 : 0, (int)o.top_k, o.top_p, o.temperature};
}
SampleCfg sub_cfg(const qtts_generate_options& o) {
  return SampleCfg{o.subtalker_dosample ? 1 : 0, (int)o.subtalker_top_k, o.subtalker_top_p,
                   o.subtalker_temperature};
}


std::vector<float> to_f32(const TensorRef& t);
void expect_shape(const std::string& name, const TensorRef& t, std::vector<long long> shape);

// Codec decoder (HipCodecInitial, src/audio/codec_hip.rs:203-1087): codes
// [frames x 16] -> 24 kHz waveform. Loaded from speech_tokenizer/model.safetensors
// when present; weights stay fp32 like the reference's and are packed at load
// into the layouts the kernels of codec.cu read (channel-major activations,
// every linear layer a 1x1 convolution, transposed convolutions split into
// one causal convolution per output phase).
class Codec {
 public:
  static constexpr int kGroups = 16, kCbSize = 2048, kCbDim = 256, kProj = 512, kPre = 1024;
  static constexpr int kHidden = 512, kLayers = 8, kHeads = 16, kHeadDim = 64, kInter = 1024;
  static constexpr int kUp = 1024, kCnx = 4096, kDec0 = 1536, kFinal = 96;
  static constexpr int kBlocks[4][3] = {{1536, 768, 8}, {768, 384, 5}, {384, 192, 4}, {192, 96, 3}};
  static constexpr int kDil[3] = {1, 3, 9};

  Codec(const std::string& path, cudaStream_t stream) : stream_(stream) {
    SafeTensors st(path);
    auto get = [&](const std::string& n, std::vector<long long> shape) {
      TensorRef t = st.get(n);
      expect_shape(n, t, shape);
      return to_f32(t);
    };
    auto up = [&](const std::vector<float>& v) {
      float* d = arena_.alloc<float>(v.size());
      QCK(cudaMemcpy(d, v.data(), v.size() * 4, cudaMemcpyHostToDevice));
      return d;
    };
    auto vec = [&](const std::string& n, long long len) { return up(get(n, {len})); };
    // snake: e^alpha, e^beta per channel, computed on the device with expf
    auto snake = [&](const std::string& p, int C, float** a, float** b) {
      float* ra = vec(p + ".alpha", C);
      float* rb = vec(p + ".beta", C);
      *a = arena_.alloc<float>(C);
      *b = arena_.alloc<float>(C);
      QCK(codec_exp(ra, C, *a, stream_));
      QCK(codec_exp(rb, C, *b, stream_));
    };
    // normalised codebooks (codec_hip.rs:2135-2154)
    auto book = [&](const std::string& p) {
      std::vector<float> e = get(p + "._codebook.embedding_sum", {kCbSize, kCbDim});
      std::vector<float> u = get(p + "._codebook.cluster_usage", {kCbSize});
      for (int c = 0; c < kCbSize; ++c) {
        const float sc = std::max(u[c], 1e-7f);
        for (int d = 0; d < kCbDim; ++d) e[(size_t)c * kCbDim + d] /= sc;
      }
      return e;
    };
    const std::string q = "decoder.quantizer";
    cb_first_ = up(book(q + ".rvq_first.vq.layers.0"));
    {
      std::vector<float> rest;
      for (int g = 0; g < kGroups - 1; ++g) {
        std::vector<float> b = book(q + ".rvq_rest.vq.layers." + std::to_string(g));
        rest.insert(rest.end(), b.begin(), b.end());
      }
      cb_rest_ = up(rest);
    }
    wf_ = up(get(q + ".rvq_first.output_proj.weight", {kProj, kCbDim, 1}));
    wr_ = up(get(q + ".rvq_rest.output_proj.weight", {kProj, kCbDim, 1}));
    pre_w_ = up(get("decoder.pre_conv.conv.weight", {kPre, kProj, 3}));
    pre_b_ = vec("decoder.pre_conv.conv.bias", kPre);
    const std::string t = "decoder.pre_transformer";
    in_w_ = up(get(t + ".input_proj.weight", {kHidden, kPre}));
    in_b_ = vec(t + ".input_proj.bias", kHidden);
    out_w_ = up(get(t + ".output_proj.weight", {kPre, kHidden}));
    out_b_ = vec(t + ".output_proj.bias", kPre);
    norm_ = vec(t + ".norm.weight", kHidden);
    const int qo = kHeads * kHeadDim;
    for (int l = 0; l < kLayers; ++l) {
      const std::string p = t + ".layers." + std::to_string(l);
      Layer& L = layers_[l];
      L.in_g = vec(p + ".input_layernorm.weight", kHidden);
      std::vector<float> qkv;
      for (const char* nm : {"q_proj", "k_proj", "v_proj"}) {
        std::vector<float> w = get(p + ".self_attn." + nm + ".weight", {qo, kHidden});
        qkv.insert(qkv.end(), w.begin(), w.end());
      }
      L.wqkv = up(qkv);
      L.wo = up(get(p + ".self_attn.o_proj.weight", {kHidden, qo}));
      L.attn_scale = vec(p + ".self_attn_layer_scale.scale", kHidden);
      L.post_g = vec(p + ".post_attention_layernorm.weight", kHidden);
      std::vector<float> gu = get(p + ".mlp.gate_proj.weight", {kInter, kHidden});
      std::vector<float> u = get(p + ".mlp.up_proj.weight", {kInter, kHidden});
      gu.insert(gu.end(), u.begin(), u.end());
      L.wgu = up(gu);
      L.wdown = up(get(p + ".mlp.down_proj.weight", {kHidden, kInter}));
      L.mlp_scale = vec(p + ".mlp_layer_scale.scale", kHidden);
    }
    for (int i = 0; i < 2; ++i) {
      const std::string p = "decoder.upsample." + std::to_string(i);
      Up& U = ups_[i];
      // transposed conv, kernel = stride = 2: phase p uses tap p alone
      U.tw = up(pack_trans(get(p + ".0.conv.weight", {kUp, kUp, 2}), kUp, kUp, 2, 2));
      U.tb = vec(p + ".0.conv.bias", kUp);
      U.dw = up(get(p + ".1.dwconv.conv.weight", {kUp, 1, 7}));
      U.dwb = vec(p + ".1.dwconv.conv.bias", kUp);
      U.ln_g = vec(p + ".1.norm.weight", kUp);
      U.ln_b = vec(p + ".1.norm.bias", kUp);
      U.pw1 = up(get(p + ".1.pwconv1.weight", {kCnx, kUp}));
      U.pw1b = vec(p + ".1.pwconv1.bias", kCnx);
      U.pw2 = up(get(p + ".1.pwconv2.weight", {kUp, kCnx}));
      U.pw2b = vec(p + ".1.pwconv2.bias", kUp);
      U.gamma = vec(p + ".1.gamma", kUp);
    }
    d0_w_ = up(get("decoder.decoder.0.conv.weight", {kDec0, kPre, 7}));
    d0_b_ = vec("decoder.decoder.0.conv.bias", kDec0);
    for (int b = 0; b < 4; ++b) {
      const int cin = kBlocks[b][0], cout = kBlocks[b][1], s = kBlocks[b][2];
      const std::string p = "decoder.decoder." + std::to_string(b + 1) + ".block";
      Block& B = blocks_[b];
      snake(p + ".0", cin, &B.sa, &B.sb);
      B.tw = up(pack_trans(get(p + ".1.conv.weight", {cin, cout, 2 * s}), cin, cout, 2 * s, s));
      B.tb = vec(p + ".1.conv.bias", cout);
      for (int u = 0; u < 3; ++u) {
        const std::string r = p + "." + std::to_string(u + 2);
        Res& R = B.res[u];
        snake(r + ".act1", cout, &R.a1, &R.b1);
        R.c1 = up(get(r + ".conv1.conv.weight", {cout, cout, 7}));
        R.c1b = vec(r + ".conv1.conv.bias", cout);
        snake(r + ".act2", cout, &R.a2, &R.b2);
        R.c2 = up(get(r + ".conv2.conv.weight", {cout, cout, 1}));
        R.c2b = vec(r + ".conv2.conv.bias", cout);
      }
    }
    snake("decoder.decoder.5", kFinal, &fa_, &fb_);
    f_w_ = up(get("decoder.decoder.6.conv.weight", {1, kFinal, 7}));
    f_b_ = vec("decoder.decoder.6.conv.bias", 1);
    err_ = arena_.alloc<int>(1);
    {
      // split-K workspace of the tensor-core convolutions (one partial tile
      // per SM) and the tiles' tickets
      int dev = 0, sms = 0;
      QCK(cudaGetDevice(&dev));
      QCK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
      split_.sms = sms;
      split_.max_tiles = sms;
      split_.ws_floats = (size_t)sms * 128 * 128;
      split_.ws = arena_.alloc<float>(split_.ws_floats);
      split_.tickets = arena_.alloc<unsigned>(sms);
    }
    // Tensor-core copies (bf16 hi + lo) of every convolution weight with at
    // least 64 output channels (QTTS_CODEC_TC=0: CUDA-core kernel only).
    const char* tz = std::getenv("QTTS_CODEC_TC");
    if (!(tz && tz[0] == '0') && tc_available()) {
      QCK(cudaDeviceSynchronize());  // the uploads above have landed
      auto tcw = [&](const float* w, int rows, int ci, int taps) {
        if (rows < 64) return;
        CodecTcWeight t;
        const size_t n = (size_t)rows * taps * codec_tc_padded_channels(ci);
        __nv_bfloat16* hi = arena_.alloc<__nv_bfloat16>(n);
        __nv_bfloat16* lo = arena_.alloc<__nv_bfloat16>(n);
        QCK(codec_tc_prepare(w, rows, ci, taps, hi, lo, &t, stream_));
        tc_w_[w] = t;
      };
      const int qo = kHeads * kHeadDim;
      tcw(pre_w_, kPre, kProj, 3);
      tcw(in_w_, kHidden, kPre, 1);
      tcw(out_w_, kPre, kHidden, 1);
      for (const Layer& L : layers_) {
        tcw(L.wqkv, 3 * qo, kHidden, 1);
        tcw(L.wo, kHidden, qo, 1);
        tcw(L.wgu, 2 * kInter, kHidden, 1);
        tcw(L.wdown, kHidden, kInter, 1);
      }
      for (const Up& U : ups_) {
        tcw(U.tw, 2 * kUp, kUp, 1);
        tcw(U.pw1, kCnx, kUp, 1);
        tcw(U.pw2, kUp, kCnx, 1);
      }
      tcw(d0_w_, kDec0, kPre, 7);
      for (int b = 0; b < 4; ++b) {
        const int cin = kBlocks[b][0], cout = kBlocks[b][1], s = kBlocks[b][2];
        tcw(blocks_[b].tw, s * cout, cin, 2);
        for (const Res& R : blocks_[b].res) {
          tcw(R.c1, cout, cout, 7);
          tcw(R.c2, cout, cout, 1);
        }
      }
    }
    QCK(cudaStreamSynchronize(stream_));
  }
  ~Codec() { release(); }

  static constexpr int samples_per_frame() { return 2 * 2 * 8 * 5 * 4 * 3; }
  size_t device_bytes() const { return arena_.bytes() + ws_bytes_; }

  // Carried state of a streaming decode: each causal convolution's last input
  // columns (double-buffered: a chunk reads one set and writes the other) and
  // the pre-transformer's keys / values of every decoded frame. Decoding a
  // stream chunk by chunk computes what one decode of all its frames computes.
  struct StreamState {
    int cap = 0;     // frames the stream may decode in total
    int frames = 0;  // frames decoded so far
    int cur = 0;     // which state set the next chunk reads
    std::vector<float*> st[2];
    float* kv = nullptr;  // [layers][2][heads][cap][head_dim]
    StreamState() = default;
    StreamState(const StreamState&) = delete;
    StreamState& operator=(const StreamState&) = delete;
    ~StreamState() {
      for (auto& v : st)
        for (float* p : v) cudaFree(p);
      if (kv) cudaFree(kv);
    }
  };

  // Channels and history columns of every causal convolution, in decode order.
  static std::vector<std::pair<int, int>> stream_convs() {
    std::vector<std::pair<int, int>> v;
    v.push_back({kProj, 2});  // pre_conv (3 taps)
    v.push_back({kUp, 6});    // upsample 0 dwconv (7 taps)
    v.push_back({kUp, 6});    // upsample 1 dwconv
    v.push_back({kPre, 6});   // decoder.0 (7 taps)
    for (int b = 0; b < 4; ++b) {
      v.push_back({kBlocks[b][0], 1});  // transposed convolution: inputs i - 1, i
      for (int u = 0; u < 3; ++u) v.push_back({kBlocks[b][1], 6 * kDil[u]});
    }
    v.push_back({kFinal, 6});  // decoder.6
    return v;
  }
  std::unique_ptr<StreamState> open_stream(int cap) {
    auto s = std::make_unique<StreamState>();
    s->cap = cap;
    for (auto [C, H] : stream_convs())
      for (int k = 0; k < 2; ++k) {
        void* p = nullptr;
        QCK(cudaMalloc(&p, (size_t)C * H * 4));
        QCK(cudaMemsetAsync(p, 0, (size_t)C * H * 4, stream_));
        s->st[k].push_back(static_cast<float*>(p));
      }
    void* p = nullptr;
    const size_t kvn = (size_t)kLayers * 2 * kHeads * cap * kHeadDim;
    QCK(cudaMalloc(&p, kvn * 4));
    s->kv = static_cast<float*>(p);
    QCK(cudaStreamSynchronize(stream_));
    return s;
  }

  // HipTtsEngine::decode_codes (generation.rs:619-646) for `frames` frames of
  // device-resident codes; the waveform (frames * 1920 samples) is left in
  // out() on the stream.
  void decode(const int32_t* d_codes, int frames) { run(d_codes, frames, nullptr); }
  // The next `frames` frames of a streaming decode: out() receives the
  // waveform of exactly these frames, equal to their samples in one decode
  // of the whole stream.
  void decode_chunk(StreamState& s, const int32_t* d_codes, int frames) {
    if (s.frames + frames > s.cap) throw QttsError(QTTS_ERR_INVALID_INPUT, "codec stream is full");
    run(d_codes, frames, &s);
    s.frames += frames;
    s.cur ^= 1;
  }

 private:
  void run(const int32_t* d_codes, int frames, StreamState* s) {
    ensure(frames);
    const int T = frames;
    launches = 0;
    tc_launches = 0;
    int sc = 0;  // next causal convolution's state slot
    // x with its carried history in front (ws_.cat), or x alone (one-shot)
    auto hist = [&](const float* x, int C, int n, int* h) -> const float* {
      const int slot = sc++;
      if (!s) {
        *h = 0;
        return x;
      }
      const int H = stream_convs_[slot].second;
      QCK(codec_hist_cat(s->st[s->cur][slot], x, C, H, n, ws_.cat, s->st[s->cur ^ 1][slot],
                         stream_));
      ++launches;
      *h = H;
      return ws_.cat;
    };
    int h = 0;
    const int pos0 = s ? s->frames : 0, kvcap = s ? s->cap : T;
    // RVQ + pre_conv
    QCK(codec_rvq(d_codes, T, kGroups, kCbSize, kCbDim, cb_first_, cb_rest_, wf_, wr_, kProj,
                  ws_.first, ws_.rest, ws_.a, stream_));
    launches += 2;
    const float* xin = hist(ws_.a, kProj, T, &h);
    conv(xin, kProj, T, pre_w_, 0, pre_b_, kPre, 3, 1, 2, ws_.b, h);
    // pre_transformer (codec_hip.rs:379-653)
    conv(ws_.b, kPre, T, in_w_, 0, in_b_, kHidden, 1, 1, 0, ws_.h);
    const int qo = kHeads * kHeadDim;
    for (int l = 0; l < kLayers; ++l) {
      const Layer& L = layers_[l];
      float* kc = s ? s->kv + (size_t)l * 2 * kHeads * kvcap * kHeadDim : ws_.k;
      float* vc = s ? kc + (size_t)kHeads * kvcap * kHeadDim : ws_.v;
      QCK(codec_chan_norm(ws_.h, kHidden, T, L.in_g, nullptr, 1e-5f, ws_.n, stream_));
      conv(ws_.n, kHidden, T, L.wqkv, 0, nullptr, 3 * qo, 1, 1, 0, ws_.qkv);
      QCK(codec_qkv_rope(ws_.qkv, kHeads, kHeadDim, T, pos0, kvcap, 10000.0f, ws_.q, kc, vc,
                         stream_));
      QCK(codec_attention(ws_.q, kc, vc, kHeads, kHeadDim, T, pos0, kvcap,
                          1.0f / std::sqrt(64.0f), ws_.att, stream_));
      launches += 3;
      conv(ws_.att, qo, T, L.wo, 0, nullptr, kHidden, 1, 1, 0, ws_.h, 0, CACT_NONE, nullptr,
           nullptr, 0, CEPI_RESID, ws_.h, L.attn_scale);
      QCK(codec_chan_norm(ws_.h, kHidden, T, L.post_g, nullptr, 1e-5f, ws_.n, stream_));
      ++launches;
      conv(ws_.n, kHidden, T, L.wgu, 0, nullptr, 2 * kInter, 1, 1, 0, ws_.qkv);
      conv(ws_.qkv, kInter, T, L.wdown, 0, nullptr, kHidden, 1, 1, 0, ws_.h, 0, CACT_SWIGLU,
           nullptr, nullptr, kInter, CEPI_RESID, ws_.h, L.mlp_scale);
    }
    QCK(codec_chan_norm(ws_.h, kHidden, T, norm_, nullptr, 1e-5f, ws_.n, stream_));
    ++launches;
    conv(ws_.n, kHidden, T, out_w_, 0, out_b_, kPre, 1, 1, 0, ws_.a);
    // upsample stages (codec_hip.rs:656-785)
    float* x = ws_.a;
    int L = T;
    for (int i = 0; i < 2; ++i) {
      const Up& U = ups_[i];
      float* y = x == ws_.a ? ws_.b : ws_.a;
      conv(x, kUp, L, U.tw, (long long)kUp * kUp, U.tb, kUp, 1, 1, 0, y, 0, CACT_NONE, nullptr,
           nullptr, 0, 0, nullptr, nullptr, 2, 2);
      L *= 2;
      const float* yin = hist(y, kUp, L, &h);
      QCK(codec_dwconv(yin, kUp, L, h, U.dw, U.dwb, 7, ws_.n, stream_));
      QCK(codec_chan_norm(ws_.n, kUp, L, U.ln_g, U.ln_b, 1e-6f, ws_.att, stream_));
      launches += 2;
      conv(ws_.att, kUp, L, U.pw1, 0, U.pw1b, kCnx, 1, 1, 0, ws_.qkv, 0, CACT_NONE, nullptr,
           nullptr, 0, CEPI_GELU);
      conv(ws_.qkv, kCnx, L, U.pw2, 0, U.pw2b, kUp, 1, 1, 0, y, 0, CACT_NONE, nullptr, nullptr, 0,
           CEPI_RESID, y, U.gamma);
      x = y;
    }
    // decoder (codec_hip.rs:787-1041). Every snake is applied once, in the
    // epilogue of the convolution that produces its input: decoder.0 stores
    // snake(y) for block 0; a transposed convolution stores the residual
    // stream x and snake(x) for its first residual unit; conv1 stores
    // snake2(y); conv2 updates x in place and stores snake(x) for whatever
    // reads it next (the next unit, the next block, the final convolution).
    float* s_in = ws_.sa;
    float* s_out = ws_.sb;
    xin = hist(x, kPre, L, &h);
    conv(xin, kPre, L, d0_w_, 0, d0_b_, kDec0, 7, 1, 6, s_in, h, CACT_NONE, nullptr, nullptr, 0,
         CEPI_SNAKE, nullptr, nullptr, 1, 1, blocks_[0].sa, blocks_[0].sb);
    for (int b = 0; b < 4; ++b) {
      const int cin = kBlocks[b][0], cout = kBlocks[b][1], st = kBlocks[b][2];
      const Block& B = blocks_[b];
      xin = hist(s_in, cin, L, &h);
      conv(xin, cin, L, B.tw, (long long)cout * cin * 2, B.tb, cout, 2, 1, 1, ws_.x, h, CACT_NONE,
           nullptr, nullptr, 0, 0, nullptr, nullptr, st, st, B.res[0].a1, B.res[0].b1, s_out);
      L *= st;
      for (int u = 0; u < 3; ++u) {
        const Res& R = B.res[u];
        xin = hist(s_out, cout, L, &h);
        conv(xin, cout, L, R.c1, 0, R.c1b, cout, 7, kDil[u], 6 * kDil[u], ws_.scr, h, CACT_NONE,
             nullptr, nullptr, 0, CEPI_SNAKE, nullptr, nullptr, 1, 1, R.a2, R.b2);
        const float* na = u < 2 ? B.res[u + 1].a1 : b < 3 ? blocks_[b + 1].sa : fa_;
        const float* nb = u < 2 ? B.res[u + 1].b1 : b < 3 ? blocks_[b + 1].sb : fb_;
        conv(ws_.scr, cout, L, R.c2, 0, R.c2b, cout, 1, 1, 0, ws_.x, 0, CACT_NONE, nullptr,
             nullptr, 0, CEPI_RESID, ws_.x, nullptr, 1, 1, na, nb, s_out);
      }
      std::swap(s_in, s_out);
    }
    xin = hist(s_in, kFinal, L, &h);
    conv(xin, kFinal, L, f_w_, 0, f_b_, 1, 7, 1, 6, ws_.wav, h, CACT_NONE, nullptr, nullptr, 0,
         CEPI_CLAMP);
  }

 public:
  const float* out() const { return ws_.wav; }
  size_t launches = 0;     // kernels enqueued by the last decode
  size_t tc_launches = 0;  // of which tensor-core convolutions
  // Throws if a tensor-core convolution reported a pipeline timeout (call
  // after the stream has drained); the status is cleared.
  void check_status() {
    int e = 0;
    QCK(cudaMemcpy(&e, err_, sizeof e, cudaMemcpyDeviceToHost));
    if (e) {
      QCK(cudaMemset(err_, 0, sizeof e));
      throw QttsError(QTTS_ERR_CUDA, "codec tensor-core convolution: pipeline wait " +
                                         std::to_string(e) + " timed out");
    }
  }
  int32_t* codes_buffer(int frames) {
    ensure(frames);
    return ws_.codes;
  }

 private:
  struct Layer {
    float *in_g, *wqkv, *wo, *attn_scale, *post_g, *wgu, *wdown, *mlp_scale;
  } layers_[kLayers]{};
  struct Up {
    float *tw, *tb, *dw, *dwb, *ln_g, *ln_b, *pw1, *pw1b, *pw2, *pw2b, *gamma;
  } ups_[2]{};
  struct Res {
    float *a1, *b1, *c1, *c1b, *a2, *b2, *c2, *c2b;
  };
  struct Block {
    float *sa, *sb, *tw, *tb;
    Res res[3];
  } blocks_[4]{};
  struct Ws {
    int32_t* codes;
    float *first, *rest, *a, *b, *h, *n, *qkv, *q, *k, *v, *att, *x, *sa, *sb, *scr, *wav, *cat;
  } ws_{};
  const std::vector<std::pair<int, int>> stream_convs_ = stream_convs();

  // Transposed convolution weight [cin][cout][K] (stride s, K = s or 2 s)
  // as one causal convolution per output phase p: [p][cout][cin * taps],
  // taps ordered oldest input first (tap 0 reads input i - 1 through
  // W[.][.][p + s] when K = 2 s, the last tap reads input i through W[.][.][p]).
  static std::vector<float> pack_trans(const std::vector<float>& w, int cin, int cout, int K,
                                       int s) {
    const int taps = K / s;
    std::vector<float> o((size_t)s * cout * cin * taps);
    for (int p = 0; p < s; ++p)
      for (int co = 0; co < cout; ++co)
        for (int ci = 0; ci < cin; ++ci)
          for (int j = 0; j < taps; ++j) {
            const int k = p + (taps - 1 - j) * s;
            o[(((size_t)p * cout + co) * cin + ci) * taps + j] =
                w[((size_t)ci * cout + co) * K + k];
          }
    return o;
  }

  void conv(const float* x, int ci, int lin, const float* w, long long w_phase_stride,
            const float* bias, int co, int taps, int dil, int pad, float* y, int hist = 0,
            int act = CACT_NONE,
            const float* act_a = nullptr, const float* act_b = nullptr, int up_off = 0,
            int epi = 0, const float* resid = nullptr, const float* rscale = nullptr,
            int ostride = 1, int nphase = 1, const float* out_a = nullptr,
            const float* out_b = nullptr, float* y2 = nullptr) {
    CodecConvArgs a{x,   ci,     lin,    w,      w_phase_stride, bias,  co,     taps, dil,
                    pad, act,    act_a,  act_b,  up_off,         y,     ostride, nphase, epi,
                    resid, rscale, out_a, out_b, y2, hist};
    auto it = tc_w_.find(w);
    if (it != tc_w_.end() && codec_tc_supported(a, it->second)) {
      QCK(codec_conv_tc(a, it->second, err_, &split_, stream_));
      ++tc_launches;
    } else {
      QCK(codec_conv(a, stream_));
    }
    ++launches;
  }

  void ensure(int frames) {
    if (frames <= cap_) return;
    release();
    const size_t T = (size_t)frames;
    size_t big = 0;  // largest decoder activation per frame, in floats
    {
      size_t L = 4;  // decoder input steps per frame (after the two upsample stages)
      big = std::max(big, (size_t)kDec0 * L);
      for (int b = 0; b < 4; ++b) {
        L *= kBlocks[b][2];
        big = std::max(big, (size_t)kBlocks[b][1] * L);
      }
      big = std::max(big, L);
    }
    auto al = [&](size_t n) {
      void* p = nullptr;
      QCK(cudaMalloc(&p, std::max<size_t>(n, 4) * 4));
      ws_bytes_ += std::max<size_t>(n, 4) * 4;
      return static_cast<float*>(p);
    };
    const int qo = kHeads * kHeadDim;
    ws_.codes = reinterpret_cast<int32_t*>(al(T * kGroups));
    ws_.first = al(T * kCbDim);
    ws_.rest = al(T * kCbDim);
    ws_.a = al(T * 4 * kUp);
    ws_.b = al(T * 4 * kUp);
    ws_.h = al(T * kHidden);
    ws_.n = al(T * 4 * kUp);
    ws_.qkv = al(T * std::max(3 * qo, 4 * kCnx));
    ws_.q = al(T * qo);
    ws_.k = al(T * qo);
    ws_.v = al(T * qo);
    ws_.att = al(T * 4 * kUp);
    ws_.x = al(T * big);
    ws_.sa = al(T * big);
    ws_.sb = al(T * big);
    ws_.scr = al(T * big);
    ws_.wav = al(T * samples_per_frame());
    // a streamed convolution's input with its history in front
    size_t hist_max = 0;
    for (auto [C, H] : stream_convs_) hist_max = std::max(hist_max, (size_t)C * H);
    ws_.cat = al(T * std::max(big, (size_t)4 * kUp) + hist_max);
    cap_ = frames;
  }
  void release() {
    for (float* p : {reinterpret_cast<float*>(ws_.codes), ws_.first, ws_.rest, ws_.a, ws_.b, ws_.h,
                     ws_.n, ws_.qkv, ws_.q, ws_.k, ws_.v, ws_.att, ws_.x, ws_.sa, ws_.sb,
                     ws_.scr, ws_.wav, ws_.cat})
      if (p) cudaFree(p);
    ws_ = Ws{};
    ws_bytes_ = 0;
    cap_ = 0;
  }

  cudaStream_t stream_;
  Arena arena_;
  float *cb_first_ = nullptr, *cb_rest_ = nullptr, *wf_ = nullptr, *wr_ = nullptr;
  float *pre_w_ = nullptr, *pre_b_ = nullptr, *in_w_ = nullptr, *in_b_ = nullptr;
  float *out_w_ = nullptr, *out_b_ = nullptr, *norm_ = nullptr;
  float *d0_w_ = nullptr, *d0_b_ = nullptr, *fa_ = nullptr, *fb_ = nullptr, *f_w_ = nullptr,
        *f_b_ = nullptr;
  int cap_ = 0;
  size_t ws_bytes_ = 0;
  int* err_ = nullptr;  // tensor-core pipeline status (nonzero: a wait ran out)
  CodecTcSplit split_;
  std::unordered_map<const float*, CodecTcWeight> tc_w_;
};

class Engine {
 public:
  Engine(const std::string& dir, int device, const qtts_cache_options& cache);
  ~Engine();

  // How the talker's cache is kept: bf16 with every position seen, by the fused
  // decode and prefill attention of kernels.cu; or in 4 bits and / or seen
  // through a window, by the kernels of kv_*.cu (kv_form).
  const qtts_cache_options cache;
  bool kv_form() const { return cache.kv_bits != 16 || cache.window != 0; }
  int* kv_word = nullptr;  // their status
  KvArgs kv_args(const KvView& kv, int seqs, int max_pages, const int* pos, int pos_stride, int pos0);
  void kv_attention(DevStack& S, StackBufs& B, const KvArgs& c, const KvRows& r, int layer,
                    const int* halt, int halt_stride);
  void check_kv();

  ModelCfg cfg;
  size_t max_cache_steps;
  int device;
  cudaStream_t stream = nullptr;
  Arena arena;

  // weights
  DevStack talker, cp;
  __nv_bfloat16 *head = nullptr, *codec_emb = nullptr, *text_emb = nullptr;
  __nv_bfloat16 *fc1 = nullptr, *fc2 = nullptr, *cp_heads = nullptr, *cp_embs = nullptr;
  __nv_bfloat16* proj_w = nullptr;
  float *norm_g = nullptr, *fc1_b = nullptr, *fc2_b = nullptr, *cp_norm_g = nullptr,
        *proj_b = nullptr;
  int text_vocab = 0, text_hidden = 0, text_inter = 0;

  // workspaces
  StackBufs tb{}, cb{};
  KvView tkv{}, ckv{};
  float *logits = nullptr, *dbg_logits = nullptr;
  unsigned* tickets = nullptr;
  SeqState* st = nullptr;
  SeqState* st_host = nullptr;  // pinned
  // Host-to-device uploads go through this pinned staging area as
  // cudaMemcpyAsync on `stream`, so the kernels that read the data are
  // ordered after the copy by the stream itself (a synchronous cudaMemcpy from
  // pageable memory may return before its DMA lands, and the non-blocking
  // engine stream does not wait for the legacy stream). Sized at load; never
  // grows, so uploads allocate nothing.
  char* stage = nullptr;
  size_t stage_cap = 0, stage_off = 0;
  void h2d(void* dst, const void* src, size_t bytes);
  void stream_sync() {
    QCK(cudaStreamSynchronize(stream));
    stage_off = 0;
  }
  int *codes = nullptr, *history = nullptr, *token = nullptr;
  float *trailing = nullptr, *tts_pad = nullptr, *cp_prefix = nullptr, *cp_next = nullptr,
        *emb_sum = nullptr, *xvec = nullptr;
  int *tp_ids = nullptr, *tp_pidx = nullptr, *tp_cids = nullptr;
  float *tp_a = nullptr, *tp_b = nullptr, *tp_c = nullptr;
  int tp_rows = 0;
  std::vector<int> pinned_ids_storage;

  std::map<SampleKey, cudaGraphExec_t> graphs;
  unsigned long long* selftest_ctr = nullptr;  // qtts_selftest_device_wait
  int* selftest_status = nullptr;
  // tcgen05 projections for M >= tc_min_rows rows (QTTS_TC=0 disables)
  // Which projections use it is fixed per call site, not per row count, so a
  // row gets identical arithmetic however the rows are batched (one-shot vs
  // streamed prompts): the talker prefill and the text MLP always, the
  // CodePredictor's 2-row prefill only with QTTS_TC_CP=1.
  TcPlan tc{};  // tokens == 0: unavailable
  int* tc_err = nullptr;
  bool tc_scope = false;
  bool tc_cp = false;
  struct TcScope {
    bool& f;
    bool old;
    TcScope(bool& flag, bool on) : f(flag), old(flag) { f = on; }
    ~TcScope() { f = old; }
  };
  // CodePredictor attention inside the O projection (QTTS_FUSE_ATTN_O=0: separate kernels)
  bool fuse_attn_o = true;
  // Layer-0 projections of every CodePredictor input token (groups 1..14 take
  // the previous group's token embedding as their input, so its QKV row depends
  // on the token alone): [groups-2][vocab][qkv_w], computed at load with the
  // tensor-core GEMM; the heads copy the selected row (and, for models with
  // the CodePredictor input projection, the projected input row, cp_x0).
  // Off with QTTS_CP_QKV_TABLE=0.
  float* cp_qkv0 = nullptr;
  float* cp_x0 = nullptr;  // with the input projection: [groups-2][vocab][cp hidden] projected rows
  void build_cp_qkv_table();
  // Talker pages in the cache's format (16 bits: page_stride elements each).
  __nv_bfloat16* alloc_talker_pool(int pages) {
    if (cache.kv_bits == 16) return arena.alloc<__nv_bfloat16>((size_t)(tkv.page_stride * pages));
    const KvGeom g{1, 1, 1, cfg.talker.layers, cfg.talker.kv_heads, kTalkerPageShift, cache.kv_bits};
    return reinterpret_cast<__nv_bfloat16*>(
        arena.alloc<unsigned char>((size_t)kv_page_bytes(g) * pages));
  }
  cudaEvent_t ev0 = nullptr, ev1 = nullptr, ev2 = nullptr;
  float last_prefill_ms = 0.f, last_frames_ms = 0.f;
  size_t last_frames = 0;
  size_t launches = 0;        // kernels enqueued directly (or captured) by this engine
  size_t last_launches = 0;   // kernels launched by the last generation (graphs expanded)
  std::map<SampleKey, size_t> graph_nodes;

  // current sequence (host view)
  int seq_P = 0;
  int seq_frames = 0;
  int seq_semantic = -1;
  bool seq_ended = false;
  size_t seq_max_frames = 0;
  qtts_generate_options seq_opts{};
  // codec decoder (speech_tokenizer/model.safetensors); null when absent
  std::unique_ptr<Codec> codec;
  size_t decode_codes(const int32_t* codes, size_t n_codes, float* out, size_t cap,
                      Codec::StreamState* cs = nullptr);
  float last_decode_ms = 0.f;  // device time of the last decode (codes resident to waveform)
  uint64_t seq_id = 0;

  bool has_proj() const { return cfg.cp.hidden != cfg.talker.hidden; }
  float* cp_prefix_target() const { return has_proj() ? cp_prefix : cb.x; }
  float* cp_next_target() const { return has_proj() ? cp_next : cb.x; }

  // ---- launch helpers ----
  void linear(const __nv_bfloat16* W, const float* x, int ldx, const float* gamma, float eps,
              float* y, int ldy, const float* resid, int ldr, const float* bias, int M, int N,
              int K, Epilogue epi, const int* halt, bool resid_early = false) {
    LinearArgs a{W, x, ldx, gamma, eps, y, ldy, resid, ldr, bias, M, N, K, halt};
    a.resid_early = resid_early;
    if (tc_scope && tc.tokens && tc_supported(a, epi, tc)) {
      QCK(launch_linear_tc(a, epi, tc, nullptr, tc_err, stream));  // tcgen05 GEMM
      launches += 1;
      return;
    }
    static const char* kEpi[] = {"gemv", "gemv+resid", "gemv+swiglu", "gemv+bias", "gemv+bias+silu"};
    a.trace_id = trace_tag(kEpi[epi], N, K);
    QCK(launch_linear(a, epi, stream));
    ++launches;
  }

  // Post-attention half of a decode layer for one row: B.x = B.h1 + MLP(B.h1).
  void mlp(const DevStack& S, int l, StackBufs& B, const int* halt) {
    const StackCfg& c = S.c;
    linear(S.wgu[l], B.h1, c.hidden, S.post_g[l], c.eps, B.act, c.intermediate, nullptr, 0,
           nullptr, 1, c.intermediate, c.hidden, EPI_SWIGLU, halt);
    // B.h1 comes from the O projection, two launches back
    linear(S.wdown[l], B.act, c.intermediate, nullptr, 0.f, B.x, c.hidden, B.h1, c.hidden,
           nullptr, 1, c.hidden, c.intermediate, EPI_RESID, halt, true);
  }

  // ---- step trace (QTTS_STEP_TRACE=<file>, or qtts_step_trace_enable) ----
  // Frame `trace_frame` of each run records, per launch, the first CTA entry,
  // the first CTA past its dependency wait and the last CTA exit.
  std::string step_trace_path;
  unsigned long long* step_trace = nullptr;
  static constexpr int kTraceCap = 4096;
  bool trace_on = false;
  std::vector<qtts_trace_launch> trace_rows;  // the last traced frame
  bool trace_capture = false;
  std::vector<std::string> trace_names;
  size_t trace_frame = 6;
  int trace_tag(const char* kind, int N, int K) {
    if (!trace_capture || (int)trace_names.size() + 1 >= kTraceCap) return 0;
    trace_names.push_back(std::string(kind) + " N=" + std::to_string(N) + " K=" + std::to_string(K));
    return (int)trace_names.size();
  }
  void dump_step_trace();

  unsigned* crumbs_host = nullptr;  // QTTS_CRUMBS=1: last kernel ids entered / left
  void stack_rows(DevStack& S, StackBufs& B, const KvView& kv, int M, int pos0, const int* halt);
  void stack_step(DevStack& S, StackBufs& B, const KvView& kv, const int* pos_ptr, int pos_const,
                  const int* halt, bool qkv0_given = false);
  HeadArgs head_args(int role, const SampleCfg& c, const int* halt);
  void talker_head(int role, const float* x, const SampleCfg& c, float penalty, const int* halt,
                   float* cp_prefix_dst);
  void cp_head(int group, const float* x, const SampleCfg& c, const int* halt);
  void enqueue_frame(const SampleKey& k);

  // ---- batched serving: up to kBatchCap sequences stepped in lockstep ----
  // Each request is prefilled alone (the validated single-sequence path,
  // writing into its own slot of the batch KV pool), then every frame runs
  // the CodePredictor pass and the talker step for all sequences at once:
  // projections as tcgen05 GEMMs with M = B (weights read once per frame for
  // the whole batch), attention and token selection per sequence.
  static constexpr int kBatchCap = 16;
  struct BatchBufs {
    int cap = 0;
    SeqState* st = nullptr;
    SeqState* st_host = nullptr;
    int *codes = nullptr, *history = nullptr;
    float *trailing = nullptr, *cp_prefix = nullptr, *cp_next = nullptr, *emb_sum = nullptr,
          *logits = nullptr;
    StackBufs tb{}, cb{};
    KvView tkv{}, ckv{};
    int pages = 0;  // talker KV pages per sequence
    // takes of one prompt: tables of their own over tkv's pages, filled by
    // launch_kv_resize / launch_kv_fork, so that full prompt pages are shared
    KvArgs takes{};
    TcPlan plan{};
    float* rms = nullptr;  // [cap] RMS scale of each head input row
    cudaEvent_t ev[3] = {nullptr, nullptr, nullptr};  // prefill start, frames start, end
  } bt;
  // by sampling, sequences (negative: takes, on their own tables)
  std::map<std::pair<SampleKey, int>, cudaGraphExec_t> batch_graphs;
  std::map<std::pair<SampleKey, int>, size_t> batch_nodes;
  void ensure_batch();
  void blinear(const __nv_bfloat16* W, const float* x, int ldx, const float* gamma, float eps,
               float* y, int ldy, const float* resid, int ldr, const float* bias, int M, int N,
               int K, Epilogue epi, float* rms_out = nullptr);
  void batch_stack_step(DevStack& S, StackBufs& B, const KvView& kv, int pt_stride,
                        const int* pos_ptr, int pos_const, int nb, bool qkv0_given = false);
  void batch_head(int role, int group, const float* x, const SampleCfg& c, float penalty, int nb);
  void enqueue_batch_frame(const SampleKey& k, int nb, const KvView& tkv);
  cudaGraphExec_t batch_graph(const SampleKey& k, int nb, const KvView& tkv, bool takes);
  void store_slot(int b, int ntr);
  void run_batch(int nb, const qtts_generate_options& o, const KvView& view, bool takes,
                 int32_t* codes_out, size_t cap_per_request, size_t* frames_out,
                 int32_t* ended_out);
  void ensure_takes();
  void generate_takes(const uint32_t* ids, size_t n, const qtts_generate_options& o,
                      const std::vector<uint64_t>& seeds, int32_t* codes_out,
                      size_t cap_per_take, size_t* frames_out, int32_t* ended_out);
  void generate_batch(const std::vector<std::vector<uint32_t>>& ids,
                      const std::vector<qtts_generate_options>& opts, int32_t* codes_out,
                      size_t cap_per_request, size_t* frames_out, int32_t* ended_out);
  cudaGraphExec_t frame_graph(const SampleKey& k);

  // ---- text prep ----
  void project_text(const std::vector<int>& ids, float* out);
  int prepare(const uint32_t* ids, size_t n, size_t lookahead, const char* speaker,
              const char* language, const float* xvec_host, int* n_trailing);
  void check_ids(const uint32_t* ids, size_t n);

  // ---- sequence ----
  void validate(const qtts_generate_options& o) const;
  void begin(int P, int n_trailing, const qtts_generate_options& o);
  size_t run_frames(size_t n);
  void read_codes(size_t from, size_t to, int32_t* out);
  void sync_state();
};

// ---------------------------------------------------------------------------
void upload_bf16(Arena& arena, const TensorRef& t, __nv_bfloat16* dst) {
  if (t.dtype == "BF16") {
    QCK(cudaMemcpy(dst, t.data, t.nbytes, cudaMemcpyHostToDevice));
    return;
  }
  std::vector<uint16_t> tmp((size_t)t.numel());
  const float* f = reinterpret_cast<const float*>(t.data);
  for (size_t i = 0; i < tmp.size(); ++i) tmp[i] = f32_to_bf16(f[i]);
  QCK(cudaMemcpy(dst, tmp.data(), tmp.size() * 2, cudaMemcpyHostToDevice));
  (void)arena;
}

std::vector<float> to_f32(const TensorRef& t) {
  std::vector<float> out((size_t)t.numel());
  if (t.dtype == "F32") {
    std::memcpy(out.data(), t.data, t.nbytes);
  } else {
    const uint16_t* b = reinterpret_cast<const uint16_t*>(t.data);
    for (size_t i = 0; i < out.size(); ++i) out[i] = bf16_to_f32(b[i]);
  }
  return out;
}

void expect_shape(const std::string& name, const TensorRef& t, std::vector<long long> shape) {
  if (t.shape != shape) {
    std::string s = name + " shape [";
    for (size_t i = 0; i < t.shape.size(); ++i) s += (i ? "," : "") + std::to_string(t.shape[i]);
    s += "] does not match the config";
    invalid(s);
  }
}

float* upload_f32(Arena& arena, const SafeTensors& st, const std::string& name, long long n) {
  TensorRef t = st.get(name);
  expect_shape(name, t, {n});
  std::vector<float> v = to_f32(t);
  float* d = arena.alloc<float>((size_t)n);
  QCK(cudaMemcpy(d, v.data(), n * 4, cudaMemcpyHostToDevice));
  return d;
}

__nv_bfloat16* upload_matrix(Arena& arena, const SafeTensors& st, const std::string& name,
                             long long rows, long long cols) {
  TensorRef t = st.get(name);
  expect_shape(name, t, {rows, cols});
  __nv_bfloat16* d = arena.alloc<__nv_bfloat16>((size_t)(rows * cols));
  upload_bf16(arena, t, d);
  return d;
}

void load_stack(Arena& arena, const SafeTensors& st, const std::string& prefix, const StackCfg& c,
                int rope_positions, DevStack& S) {
  if (c.head_dim != kHeadDim) invalid("head_dim must be 128");
  if (c.layers <= 0) invalid("layer count must be non-zero");
  if (c.hidden % 256 != 0 || c.intermediate % 256 != 0)
    invalid("hidden and intermediate sizes must be multiples of 256");
  if (c.kv_heads <= 0 || c.q_heads % c.kv_heads != 0) invalid("q_heads must be a multiple of kv_heads");
  const int g = c.q_heads / c.kv_heads;
  if (g != 1 && g != 2 && g != 4) invalid("q_heads / kv_heads must be 1, 2 or 4");
  S.c = c;
  S.q_out = c.q_heads * c.head_dim;
  S.kv_out = c.kv_heads * c.head_dim;
  S.qkv_w = S.q_out + 2 * S.kv_out;
  const long long H = c.hidden, I = c.intermediate;
  for (int l = 0; l < c.layers; ++l) {
    const std::string p = prefix + "." + std::to_string(l);
    // One allocation per layer: [qkv rows | o | gate rows, up rows | down].
    const size_t n_qkv = (size_t)S.qkv_w * H, n_o = (size_t)H * S.q_out, n_gu = (size_t)2 * I * H,
                 n_d = (size_t)H * I;
    __nv_bfloat16* base = arena.alloc<__nv_bfloat16>(n_qkv + n_o + n_gu + n_d);
    auto put = [&](const std::string& name, long long rows, long long cols, __nv_bfloat16* dst) {
      TensorRef t = st.get(name);
      expect_shape(name, t, {rows, cols});
      upload_bf16(arena, t, dst);
    };
    put(p + ".self_attn.q_proj.weight", S.q_out, H, base);
    put(p + ".self_attn.k_proj.weight", S.kv_out, H, base + (size_t)S.q_out * H);
    put(p + ".self_attn.v_proj.weight", S.kv_out, H, base + (size_t)(S.q_out + S.kv_out) * H);
    put(p + ".self_attn.o_proj.weight", H, S.q_out, base + n_qkv);
    put(p + ".mlp.gate_proj.weight", I, H, base + n_qkv + n_o);
    put(p + ".mlp.up_proj.weight", I, H, base + n_qkv + n_o + (size_t)I * H);
    put(p + ".mlp.down_proj.weight", H, I, base + n_qkv + n_o + n_gu);
    S.wqkv.push_back(base);
    S.wo.push_back(base + n_qkv);
    S.wgu.push_back(base + n_qkv + n_o);
    S.wdown.push_back(base + n_qkv + n_o + n_gu);
    S.in_g.push_back(upload_f32(arena, st, p + ".input_layernorm.weight", H));
    S.post_g.push_back(upload_f32(arena, st, p + ".post_attention_layernorm.weight", H));
    S.q_g.push_back(upload_f32(arena, st, p + ".self_attn.q_norm.weight", c.head_dim));
    S.k_g.push_back(upload_f32(arena, st, p + ".self_attn.k_norm.weight", c.head_dim));
  }
  // RoPE table: angle = pos / powf(theta, 2i/d) in fp32 (kernels.rs:64-67).
  std::vector<float> cs((size_t)rope_positions * 64), sn((size_t)rope_positions * 64);
  for (int p = 0; p < rope_positions; ++p)
    for (int i = 0; i < 64; ++i) {
      const float expo = (float)(i * 2) / (float)c.head_dim;
      const float ang = (float)p / powf(c.theta, expo);
      cs[(size_t)p * 64 + i] = cosf(ang);
      sn[(size_t)p * 64 + i] = sinf(ang);
    }
  S.rope_cos = arena.alloc<float>(cs.size());
  S.rope_sin = arena.alloc<float>(sn.size());
  QCK(cudaMemcpy(S.rope_cos, cs.data(), cs.size() * 4, cudaMemcpyHostToDevice));
  QCK(cudaMemcpy(S.rope_sin, sn.data(), sn.size() * 4, cudaMemcpyHostToDevice));
}

StackBufs alloc_bufs(Arena& arena, const DevStack& S, int rows) {
  StackBufs b;
  const size_t H = S.c.hidden, I = S.c.intermediate;
  b.x = arena.alloc<float>(rows * H);
  b.qkv = arena.alloc<float>((size_t)rows * S.qkv_w);
  b.q = arena.alloc<float>((size_t)rows * S.q_out);
  b.attn = arena.alloc<float>((size_t)rows * S.q_out);
  b.h1 = arena.alloc<float>(rows * H);
  b.act = arena.alloc<float>(rows * I);
  return b;
}

Engine::Engine(const std::string& dir, int dev, const qtts_cache_options& co)
    : cache(co), max_cache_steps(co.max_cache_steps), device(dev) {
  const size_t mcs = max_cache_steps;
  if (mcs == 0) invalid("max_cache_steps must be non-zero");
  if (co.kv_bits != 16 && co.kv_bits != 4)
    invalid("kv_bits must be 16 or 4, got " + std::to_string(co.kv_bits));
  if (co.window < 0 || co.sinks < 0) invalid("window and sinks must not be negative");
  if (co.sinks > 0 && co.window == 0) invalid("sinks need a window");
  cfg = load_config(dir);
  int ndev = 0;
  QCK(cudaGetDeviceCount(&ndev));
  if (dev < 0 || dev >= ndev) invalid("device " + std::to_string(dev) + " not present");
  QCK(cudaSetDevice(dev));
  QCK(configure_kernels());
  QCK(configure_tc_kernels());
  QCK(configure_codec_tc());
  QCK(cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking));
  QCK(cudaEventCreate(&ev0));
  QCK(cudaEventCreate(&ev1));
  QCK(cudaEventCreate(&ev2));
  const StackCfg& T = cfg.talker;
  const StackCfg& C = cfg.cp;
  if (C.groups < 2) invalid("CodePredictor needs at least one semantic and one acoustic group");
  if (T.groups != C.groups) invalid("talker and CodePredictor num_code_groups differ");
  if (T.vocab > max_sample_vocab() || C.vocab > max_sample_vocab())
    invalid("vocab larger than the sampler supports");
  if (T.vocab <= 1024) invalid("talker vocab must exceed the 1024 suppressed control ids");
  if (T.hidden > 2048) invalid("talker hidden sizes above 2048 are not supported");

  SafeTensors sf(dir + "/model.safetensors");
  const SafeTensors& st_ = sf;
  load_stack(arena, st_, "talker.model.layers", T, (int)mcs, talker);
  load_stack(arena, st_, "talker.code_predictor.model.layers", C, C.groups, cp);
  norm_g = upload_f32(arena, st_, "talker.model.norm.weight", T.hidden);
  head = upload_matrix(arena, st_, "talker.codec_head.weight", T.vocab, T.hidden);
  codec_emb = upload_matrix(arena, st_, "talker.model.codec_embedding.weight", T.vocab, T.hidden);
  {
    TensorRef te = st_.get("talker.model.text_embedding.weight");
    if (te.shape.size() != 2 || (te.shape[1] != T.hidden && te.shape[1] != 2048))
      invalid("talker.model.text_embedding.weight shape; expected [vocab, text_hidden]");
    text_vocab = (int)te.shape[0];
    text_hidden = (int)te.shape[1];
    text_emb = arena.alloc<__nv_bfloat16>((size_t)te.numel());
    upload_bf16(arena, te, text_emb);
    TensorRef f1 = st_.get("talker.text_projection.linear_fc1.weight");
    if (f1.shape.size() != 2 || f1.shape[1] != text_hidden)
      invalid("invalid text projection shapes");
    text_inter = (int)f1.shape[0];
    if (text_inter % 256 != 0 || text_hidden % 256 != 0)
      invalid("text projection widths must be multiples of 256");
    fc1 = upload_matrix(arena, st_, "talker.text_projection.linear_fc1.weight", text_inter,
                        text_hidden);
    fc1_b = upload_f32(arena, st_, "talker.text_projection.linear_fc1.bias", text_inter);
    fc2 = upload_matrix(arena, st_, "talker.text_projection.linear_fc2.weight", T.hidden,
                        text_inter);
    fc2_b = upload_f32(arena, st_, "talker.text_projection.linear_fc2.bias", T.hidden);
  }
  cp_norm_g = upload_f32(arena, st_, "talker.code_predictor.model.norm.weight", C.hidden);
  const int na = C.groups - 1;
  cp_heads = arena.alloc<__nv_bfloat16>((size_t)na * C.vocab * C.hidden);
  cp_embs = arena.alloc<__nv_bfloat16>((size_t)na * C.vocab * T.hidden);
  for (int g = 0; g < na; ++g) {
    const std::string hn = "talker.code_predictor.lm_head." + std::to_string(g) + ".weight";
    TensorRef h = st_.get(hn);
    expect_shape(hn, h, {C.vocab, C.hidden});
    upload_bf16(arena, h, cp_heads + (size_t)g * C.vocab * C.hidden);
    const std::string en =
        "talker.code_predictor.model.codec_embedding." + std::to_string(g) + ".weight";
    TensorRef e = st_.get(en);
    expect_shape(en, e, {C.vocab, T.hidden});
    upload_bf16(arena, e, cp_embs + (size_t)g * C.vocab * T.hidden);
  }
  if (has_proj()) {
    proj_w = upload_matrix(arena, st_, "talker.code_predictor.small_to_mtp_projection.weight",
                           C.hidden, T.hidden);
    proj_b = upload_f32(arena, st_, "talker.code_predictor.small_to_mtp_projection.bias", C.hidden);
  }

  // workspaces
  const int rows = (int)mcs;
  {
    // split activations for the tcgen05 projections of many rows (prefill, text MLP)
    const char* tz = std::getenv("QTTS_TC");
    if (const char* tcp = std::getenv("QTTS_TC_CP")) tc_cp = tcp[0] == '1';
    if (!(tz && tz[0] == '0') && tc_available()) {
      // split-K workspace for prefill GEMMs with few 128 x 128 tiles (short prompts)
      int sms = 148;
      QCK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
      // 64-row token tiles: twice the CTAs of 128-row tiles for typical
      // prompts, half the activation conversion per stage and CTA
      tc.tokens = 64;
      if (const char* tt = std::getenv("QTTS_TC_TOKENS")) tc.tokens = std::atoi(tt);
      tc.sm_count = sms;
      tc.max_splits = 8;
      tc.ws_floats = tc_workspace_floats(128, sms);
      tc.ws = arena.alloc<float>(tc.ws_floats);
      tc.tickets = arena.alloc<unsigned>(4096);
      tc_err = arena.alloc<int>(1);
      QCK(cudaMemset(tc_err, 0, sizeof(int)));
    }
  }
  tb = alloc_bufs(arena, talker, rows);
  cb = alloc_bufs(arena, cp, 2);
  {
    const int shift = kTalkerPageShift;
    const int pages = (int)((mcs + (1u << shift) - 1) >> shift);
    tkv.page_shift = shift;
    tkv.kv_heads = T.kv_heads;
    tkv.layer_stride = (long long)2 * T.kv_heads * (1 << shift) * kHeadDim;
    tkv.page_stride = tkv.layer_stride * T.layers;
    tkv.pool = alloc_talker_pool(pages);
    std::vector<int> pt(pages);
    for (int i = 0; i < pages; ++i) pt[i] = i;
    int* d = arena.alloc<int>(pages);
    QCK(cudaMemcpy(d, pt.data(), pages * 4, cudaMemcpyHostToDevice));
    tkv.page_table = d;
  }
  {
    int shift = 0;
    while ((1 << shift) < C.groups) ++shift;
    ckv.page_shift = shift;
    ckv.kv_heads = C.kv_heads;
    ckv.layer_stride = (long long)2 * C.kv_heads * (1 << shift) * kHeadDim;
    ckv.page_stride = ckv.layer_stride * C.layers;
    ckv.pool = arena.alloc<__nv_bfloat16>((size_t)ckv.page_stride);
    ckv.page_table = arena.alloc<int>(1);  // one entry: page 0 (zeroed)
  }
  kv_word = arena.alloc<int>(1);
  logits = arena.alloc<float>(std::max(T.vocab, C.vocab));
  dbg_logits = arena.alloc<float>((size_t)na * C.vocab);
  tickets = arena.alloc<unsigned>(64);
  st = arena.alloc<SeqState>(1);
  QCK(cudaMallocHost(&st_host, sizeof(SeqState)));
  // prefill rows + trailing rows + tts_pad row, plus small id / index arrays
  stage_cap = ((2 * mcs + 4) * (size_t)T.hidden + 4 * ((size_t)mcs + 64)) * sizeof(float);
  QCK(cudaMallocHost(&stage, stage_cap));
  codes = arena.alloc<int>(mcs * C.groups);
  history = arena.alloc<int>(mcs);
  token = arena.alloc<int>(4);
  trailing = arena.alloc<float>((mcs + 1) * T.hidden);
  tts_pad = arena.alloc<float>(T.hidden);
  cp_prefix = arena.alloc<float>(2 * (size_t)T.hidden);
  cp_next = arena.alloc<float>(T.hidden);
  emb_sum = arena.alloc<float>(T.hidden);
  xvec = arena.alloc<float>(T.hidden);
  tp_rows = (int)mcs + 16;
  tp_ids = arena.alloc<int>(tp_rows);
  tp_pidx = arena.alloc<int>(tp_rows);
  tp_cids = arena.alloc<int>(tp_rows);
  tp_a = arena.alloc<float>((size_t)tp_rows * text_hidden);
  tp_b = arena.alloc<float>((size_t)tp_rows * text_inter);
  tp_c = arena.alloc<float>((size_t)tp_rows * T.hidden);
  {
    // eight slots per launch, then 16 x 16 token-selection phase stamps
    step_trace = arena.alloc<unsigned long long>(8 * (size_t)kTraceCap + 256);
    if (const char* tp = std::getenv("QTTS_STEP_TRACE")) {
      step_trace_path = tp;
      trace_on = true;
    }
    if (const char* cr = std::getenv("QTTS_CRUMBS"); cr && cr[0] == '1') {
      QCK(cudaHostAlloc(&crumbs_host, 64, cudaHostAllocMapped));
      unsigned* d = nullptr;
      QCK(cudaHostGetDevicePointer(&d, crumbs_host, 0));
      QCK(set_crumbs_kernels(d));
      QCK(set_crumbs_gemm(d));
    }
    const char* fz = std::getenv("QTTS_FUSE_ATTN_O");
    fuse_attn_o = !(fz && fz[0] == '0');
    const char* qz = std::getenv("QTTS_CP_QKV_TABLE");
    if (!(qz && qz[0] == '0') && tc.tokens) build_cp_qkv_table();
  }
  {
    // HipCodecInitial::load (codec_hip.rs:214-336); optional here so the
    // token loop also runs on talker-only checkpoints.
    const std::string cpath = dir + "/speech_tokenizer/model.safetensors";
    struct stat sb;
    if (::stat(cpath.c_str(), &sb) == 0) codec = std::make_unique<Codec>(cpath, stream);
  }
  QCK(cudaDeviceSynchronize());
}

// HipTtsEngine::decode_codes (generation.rs:619-646).
// With a codec stream state: the stream's next frames (carried state).
size_t Engine::decode_codes(const int32_t* codes, size_t n_codes, float* out, size_t cap,
                            Codec::StreamState* cs) {
  if (n_codes % Codec::kGroups != 0)
    invalid("code length " + std::to_string(n_codes) + " is not divisible by " +
            std::to_string(Codec::kGroups));
  if (n_codes == 0) return 0;
  if (!codec) fail(QTTS_ERR_UNSUPPORTED, "no codec: speech_tokenizer/model.safetensors not found");
  const size_t frames = n_codes / Codec::kGroups;
  const size_t samples = frames * Codec::samples_per_frame();
  if (samples > cap) invalid("sample buffer too small: need " + std::to_string(samples));
  if (frames > (size_t)INT32_MAX / Codec::samples_per_frame()) invalid("too many frames");
  int32_t* d = codec->codes_buffer((int)frames);
  h2d(d, codes, n_codes * sizeof(int32_t));
  QCK(cudaEventRecord(ev0, stream));
  if (cs)
    codec->decode_chunk(*cs, d, (int)frames);
  else
    codec->decode(d, (int)frames);
  QCK(cudaEventRecord(ev1, stream));
  QCK(cudaMemcpyAsync(out, codec->out(), samples * sizeof(float), cudaMemcpyDeviceToHost, stream));
  QCK(cudaStreamSynchronize(stream));
  codec->check_status();
  QCK(cudaEventElapsedTime(&last_decode_ms, ev0, ev1));
  return samples;
}

// Stream-ordered upload of `bytes` host bytes: through the pinned staging
// area when they fit (the area is reused once the stream has drained), else
// straight from the caller's memory (still ordered on the stream).
void Engine::h2d(void* dst, const void* src, size_t bytes) {
  if (bytes == 0) return;
  const size_t aligned = (bytes + 255) & ~(size_t)255;
  if (aligned > stage_cap) {
    QCK(cudaMemcpyAsync(dst, src, bytes, cudaMemcpyHostToDevice, stream));
    return;
  }
  if (stage_off + aligned > stage_cap) stream_sync();
  std::memcpy(stage + stage_off, src, bytes);
  QCK(cudaMemcpyAsync(dst, stage + stage_off, bytes, cudaMemcpyHostToDevice, stream));
  stage_off += aligned;
}

Engine::~Engine() {
  cudaSetDevice(device);
  if (stream) cudaStreamSynchronize(stream);
  for (auto& kv : graphs) cudaGraphExecDestroy(kv.second);
  for (auto& kv : batch_graphs) cudaGraphExecDestroy(kv.second);
  if (st_host) cudaFreeHost(st_host);
  if (stage) cudaFreeHost(stage);
  if (bt.st_host) cudaFreeHost(bt.st_host);
  for (auto& ev : bt.ev)
    if (ev) cudaEventDestroy(ev);
  if (ev0) cudaEventDestroy(ev0);
  if (ev1) cudaEventDestroy(ev1);
  if (ev2) cudaEventDestroy(ev2);
  if (stream) cudaStreamDestroy(stream);
}

// The talker cache as the kv_*.cu kernels see it: rows' positions end at
// pos[seq * pos_stride] (null: pos0).
KvArgs Engine::kv_args(const KvView& kv, int seqs, int max_pages, const int* pos, int pos_stride,
                       int pos0) {
  KvArgs c{};
  const int pages = bt.cap && kv.pool == bt.tkv.pool ? bt.pages * bt.cap : max_pages;
  c.g = KvGeom{pages, seqs, max_pages, cfg.talker.layers, kv.kv_heads, kv.page_shift, cache.kv_bits};
  c.pool = reinterpret_cast<unsigned char*>(kv.pool);
  c.table = const_cast<int*>(kv.page_table);
  c.lengths = const_cast<int*>(pos);
  c.len_stride = pos_stride;
  c.len_add = pos ? 1 : pos0 + 1;
  c.work = kv_word;
  return c;
}

// QK-norm, RoPE and storing of the projected rows in B.qkv, then attention of
// B.q into B.attn (decode_step_layer_on_stream / prefill_forward's attention).
void Engine::kv_attention(DevStack& S, StackBufs& B, const KvArgs& c, const KvRows& r, int layer,
                          const int* halt, int halt_stride) {
  const StackCfg& k = S.c;
  KvPrep p{B.qkv, S.qkv_w, k.q_heads, S.q_g[layer], S.k_g[layer], k.eps, S.rope_cos, S.rope_sin,
           B.q,   layer,   halt,      halt_stride};
  QCK(launch_kv_prep(c, r, p, stream));
  KvAttend a{};
  a.q = KvTensor{B.q, S.q_out, kKvDim};
  a.out = KvTensor{B.attn, S.q_out, kKvDim};
  a.type = KV_F32;
  a.q_heads = k.q_heads;
  a.scale = 1.0f / std::sqrt((float)k.head_dim);
  a.window = cache.window;
  a.sinks = cache.sinks;
  a.layer = layer;
  a.halt = halt;
  a.halt_stride = halt_stride;
  QCK(launch_kv_attend(c, r, a, stream));
  launches += 2;
}

void Engine::check_kv() {
  if (!kv_form()) return;
  int e = 0;
  QCK(cudaMemcpy(&e, kv_word, sizeof(int), cudaMemcpyDeviceToHost));
  if (!e) return;
  QCK(cudaMemset(kv_word, 0, sizeof(int)));
  fail(QTTS_ERR_DEVICE_STATE, "cache attention reported status " + std::to_string(e));
}

// Decoder layers over M rows at positions pos0.. (prefill_forward, decode.rs:1077-1298).
void Engine::stack_rows(DevStack& S, StackBufs& B, const KvView& kv, int M, int pos0,
                        const int* halt) {
  const StackCfg& c = S.c;
  const float scale = 1.0f / std::sqrt((float)c.head_dim);
  TcScope tcs(tc_scope, &S == &talker || tc_cp);
  for (int l = 0; l < c.layers; ++l) {
    linear(S.wqkv[l], B.x, c.hidden, S.in_g[l], c.eps, B.qkv, S.qkv_w, nullptr, 0, nullptr, M,
           S.qkv_w, c.hidden, EPI_STORE, halt);
    if (&S == &talker && kv_form()) {
      const int pages = (int)((max_cache_steps + (1u << kv.page_shift) - 1) >> kv.page_shift);
      kv_attention(S, B, kv_args(kv, 1, pages, nullptr, 0, pos0 + M - 1),
                   KvRows{nullptr, nullptr, 1, M, M, pos0 + M, 1}, l, halt, 0);
    } else {
    QkPrepArgs qa{B.qkv, S.q_g[l], S.k_g[l], c.eps, S.rope_cos, S.rope_sin, kv, l, pos0, M,
                  c.q_heads, B.q, halt};
    QCK(launch_qk_prep(qa, stream));
    AttnPrefillArgs pa{B.q, kv, l, pos0, M, c.q_heads, scale, B.attn, halt};
    QCK(launch_attn_prefill(pa, stream));
    launches += 2;
    }
    linear(S.wo[l], B.attn, S.q_out, nullptr, 0.f, B.h1, c.hidden, B.x, c.hidden, nullptr, M,
           c.hidden, S.q_out, EPI_RESID, halt);
    linear(S.wgu[l], B.h1, c.hidden, S.post_g[l], c.eps, B.act, c.intermediate, nullptr, 0,
           nullptr, M, c.intermediate, c.hidden, EPI_SWIGLU, halt);
    linear(S.wdown[l], B.act, c.intermediate, nullptr, 0.f, B.x, c.hidden, B.h1, c.hidden,
           nullptr, M, c.hidden, c.intermediate, EPI_RESID, halt);
  }
}

// One position through all layers (decode_step_layer_on_stream, decode.rs:1694-1894).
// qkv0_given: layer 0's projections are already in B.qkv (a row of the
// precomputed CodePredictor table, written by the previous group's head).
void Engine::stack_step(DevStack& S, StackBufs& B, const KvView& kv, const int* pos_ptr,
                        int pos_const, const int* halt, bool qkv0_given) {
  const StackCfg& c = S.c;
  const float scale = 1.0f / std::sqrt((float)c.head_dim);
  for (int l = 0; l < c.layers; ++l) {
    if (!(l == 0 && qkv0_given))
      linear(S.wqkv[l], B.x, c.hidden, S.in_g[l], c.eps, B.qkv, S.qkv_w, nullptr, 0, nullptr, 1,
             S.qkv_w, c.hidden, EPI_STORE, halt);
    AttnDecodeArgs da{B.qkv,   S.q_g[l],  S.k_g[l], c.eps,   S.rope_cos, S.rope_sin,
                      kv,      l,         pos_ptr,  pos_const, c.q_heads, scale,
                      B.attn,  halt};
    LinearArgs o{S.wo[l], B.attn, S.q_out, nullptr, 0.f, B.h1, c.hidden, B.x, c.hidden,
                 nullptr, 1, c.hidden, S.q_out, halt};
    // The O projection's residual B.x (the layer input) was written at least
    // two launches back (previous layer's down projection, or the step input
    // before this layer's QKV), except for layer 0 of a CodePredictor group
    // whose QKV row came from the table: the preceding head wrote B.x.
    o.resid_early = !(l == 0 && qkv0_given);
    if (&S == &talker && kv_form()) {
      const int pages = (int)((max_cache_steps + (1u << kv.page_shift) - 1) >> kv.page_shift);
      kv_attention(S, B, kv_args(kv, 1, pages, pos_ptr, 1, pos_const),
                   KvRows{nullptr, nullptr, 1, 1, 1, 0, 0}, l, halt, 0);
      linear(S.wo[l], B.attn, S.q_out, nullptr, 0.f, B.h1, c.hidden, B.x, c.hidden, nullptr, 1,
             c.hidden, S.q_out, EPI_RESID, halt, o.resid_early);
    } else if (fuse_attn_o && attn_o_fusable(da, o)) {
      if (&S == &cp) da.page0 = 0;  // the CodePredictor cache is one page (page 0)
      o.trace_id = trace_tag("attn+o+resid", c.hidden, S.q_out);
      QCK(launch_attn_o(da, o, stream));  // attention inside the O projection's staging
      ++launches;
    } else {
      da.trace_id = trace_tag("attn", c.q_heads, 1);
      QCK(launch_attn_decode(da, stream));
      ++launches;
      linear(S.wo[l], B.attn, S.q_out, nullptr, 0.f, B.h1, c.hidden, B.x, c.hidden, nullptr, 1,
             c.hidden, S.q_out, EPI_RESID, halt, o.resid_early);
    }
    mlp(S, l, B, halt);
  }
}

HeadArgs Engine::head_args(int role, const SampleCfg& c, const int* halt) {
  HeadArgs a{};
  a.ticket = tickets;
  a.role = role;
  a.cfg = c;
  a.st = st;
  a.penalty = 1.0f;
  a.history = history;
  a.eos_token = cfg.codec_eos;
  a.talker_codec_emb = codec_emb;
  a.H = cfg.talker.hidden;
  a.groups = cfg.cp.groups;
  a.codes = codes;
  a.history_out = history;
  a.lin.halt = halt;
  return a;
}

void Engine::talker_head(int role, const float* x, const SampleCfg& c, float penalty,
                         const int* halt, float* cp_prefix_dst) {
  HeadArgs a = head_args(role, c, halt);
  const StackCfg& T = cfg.talker;
  a.lin = LinearArgs{head,    x,       T.hidden, norm_g,  T.eps,   logits, T.vocab,
                     nullptr, 0,       nullptr,  1,       T.vocab, T.hidden, halt};
  a.penalty = penalty;
  a.suppress = 1;
  a.cp_prefix = cp_prefix_dst;
  a.token_out = token;
  a.lin.trace_id = trace_tag("talker head+select", T.vocab, T.hidden);
  QCK(launch_head(a, stream));
  ++launches;
}

void Engine::cp_head(int group, const float* x, const SampleCfg& c, const int* halt) {
  HeadArgs a = head_args(ROLE_CP_GROUP, c, halt);
  const StackCfg& C = cfg.cp;
  a.lin = LinearArgs{cp_heads + (size_t)group * C.vocab * C.hidden,
                     x, C.hidden, cp_norm_g, C.eps, logits, C.vocab, nullptr, 0, nullptr, 1,
                     C.vocab, C.hidden, halt};
  a.group = group;
  a.last_group = C.groups - 2;
  a.cp_emb = cp_embs + (size_t)group * C.vocab * cfg.talker.hidden;
  a.cp_next = cp_next_target();
  a.emb_sum = emb_sum;
  a.step_in = tb.x;
  a.trailing = trailing;
  a.tts_pad = tts_pad;
  if (cp_qkv0 && group < C.groups - 2) {
    a.qkv_table = cp_qkv0 + (size_t)group * C.vocab * cp.qkv_w;
    a.qkv_out = cb.qkv;
    a.qkv_w = cp.qkv_w;
    if (cp_x0) {
      a.x_table = cp_x0 + (size_t)group * C.vocab * C.hidden;
      a.x_out = cb.x;
      a.x_w = C.hidden;
    }
  }
  a.lin.trace_id = trace_tag("cp head+select", C.vocab, C.hidden);
  QCK(launch_head(a, stream));
  ++launches;
}

// One frame: CodePredictor pass (code_predictor.rs:366-471) then, unless it is
// the last frame, the talker decode step and its token (generation.rs:718-740).
void Engine::enqueue_frame(const SampleKey& k) {
  const int* halt = &st->halt;
  const StackCfg& C = cfg.cp;
  const int H = cfg.talker.hidden;
  if (has_proj())
    linear(proj_w, cp_prefix, H, nullptr, 0.f, cb.x, C.hidden, nullptr, 0, proj_b, 2, C.hidden,
           H, EPI_BIAS, halt);
  stack_rows(cp, cb, ckv, 2, 0, halt);
  cp_head(0, cb.x + C.hidden, k.s, halt);
  for (int g = 1; g < C.groups - 1; ++g) {
    if (has_proj() && !cp_x0)
      linear(proj_w, cp_next, H, nullptr, 0.f, cb.x, C.hidden, nullptr, 0, proj_b, 1, C.hidden,
             H, EPI_BIAS, halt);
    stack_step(cp, cb, ckv, nullptr, g + 1, halt, cp_qkv0 != nullptr);
    cp_head(g, cb.x, k.s, halt);
  }
  if (!k.last) {
    stack_step(talker, tb, tkv, &st->talker_pos, 0, halt);
    talker_head(ROLE_TALKER_STEP, tb.x, k.t, k.penalty, halt, cp_prefix_target());
  }
}

// Layer-0 QKV rows of every CodePredictor input token: the rows of group g's
// embedding table (bf16, widened to fp32) through the input RMSNorm and the
// QKV projection of CodePredictor layer 0, one tensor-core GEMM per group.
void Engine::build_cp_qkv_table() {
  const StackCfg& C = cfg.cp;
  const int V = C.vocab, H = cfg.talker.hidden, Hc = C.hidden, W = cp.qkv_w;
  const int n = C.groups - 2;  // heads 0 .. groups-3 feed groups 1 .. groups-2
  if (n <= 0 || (!has_proj() && H != Hc)) return;
  if (W > kCpQkvTableMax || W % 4 != 0 || Hc > kCpXTableMax) return;  // widths the heads copy
  cp_qkv0 = arena.alloc<float>((size_t)n * V * W);
  if (has_proj()) cp_x0 = arena.alloc<float>((size_t)n * V * Hc);
  float* rows = arena.alloc<float>((size_t)V * H);
  int* ids = arena.alloc<int>(V);
  std::vector<int> iv(V);
  for (int i = 0; i < V; ++i) iv[i] = i;
  h2d(ids, iv.data(), (size_t)V * 4);
  TcScope tcs(tc_scope, true);
  for (int g = 0; g < n; ++g) {
    QCK(launch_gather_rows(cp_embs + (size_t)g * V * H, ids, V, H, rows, stream));
    const float* x = rows;
    if (has_proj()) {  // small_to_mtp_projection of every token (code_predictor.rs:754-817)
      float* xg = cp_x0 + (size_t)g * V * Hc;
      linear(proj_w, rows, H, nullptr, 0.f, xg, Hc, nullptr, 0, proj_b, V, Hc, H, EPI_BIAS,
             nullptr);
      x = xg;
    }
    linear(cp.wqkv[0], x, Hc, cp.in_g[0], C.eps, cp_qkv0 + (size_t)g * V * W, W, nullptr, 0,
           nullptr, V, W, Hc, EPI_STORE, nullptr);
  }
  stream_sync();
}

cudaGraphExec_t Engine::frame_graph(const SampleKey& k) {
  auto it = graphs.find(k);
  if (it != graphs.end()) return it->second;
  cudaGraph_t g = nullptr;
  const size_t before = launches;
  trace_capture = trace_on && !k.last;
  if (trace_capture) trace_names.clear();
  QCK(cudaStreamBeginCapture(stream, cudaStreamCaptureModeThreadLocal));
  try {
    enqueue_frame(k);
  } catch (...) {
    cudaStreamEndCapture(stream, &g);
    if (g) cudaGraphDestroy(g);
    launches = before;
    trace_capture = false;
    throw;
  }
  QCK(cudaStreamEndCapture(stream, &g));
  trace_capture = false;
  graph_nodes[k] = launches - before;
  launches = before;
  cudaGraphExec_t exec = nullptr;
  cudaError_t e = cudaGraphInstantiate(&exec, g, 0);
  cudaGraphDestroy(g);
  QCK(e);
  graphs[k] = exec;
  return exec;
}

// ---- text prep on the device (text.rs:571-602) ----------------------------
void Engine::check_ids(const uint32_t* ids, size_t n) {
  for (size_t i = 0; i < n; ++i)
    if ((long long)ids[i] >= text_vocab)
      invalid("text token " + std::to_string(ids[i]) + " is out of range for vocab " +
              std::to_string(text_vocab));
}

void Engine::project_text(const std::vector<int>& ids, float* out) {
  const int n = (int)ids.size();
  if (n == 0) return;
  if (n > tp_rows) invalid("too many text rows");
  h2d(tp_ids, ids.data(), (size_t)n * 4);
  QCK(launch_gather_rows(text_emb, tp_ids, n, text_hidden, tp_a, stream));
  TcScope tcs(tc_scope, true);
  linear(fc1, tp_a, text_hidden, nullptr, 0.f, tp_b, text_inter, nullptr, 0, fc1_b, n,
         text_inter, text_hidden, EPI_BIAS_SILU, nullptr);
  linear(fc2, tp_b, text_inter, nullptr, 0.f, out, cfg.talker.hidden, nullptr, 0, fc2_b, n,
         cfg.talker.hidden, text_inter, EPI_BIAS, nullptr);
}

// prepare_custom_voice_with_lookahead / prepare_voice_clone_xvector_with_lookahead
// (text.rs:348-382,432-514): writes the prefill rows into the talker input, the
// trailing rows and tts_pad row into their device buffers; returns P.
int Engine::prepare(const uint32_t* ids, size_t n, size_t lookahead, const char* speaker,
                    const char* language, const float* xvec_host, int* n_trailing) {
  check_ids(ids, n);
  const std::string spk = speaker ? speaker : "ryan";
  const std::string lang = language ? language : "english";
  auto li = cfg.language_ids.find(lang);
  if (li == cfg.language_ids.end()) invalid("missing language token id for " + lang);
  int spk_id = -2;
  if (!xvec_host) {
    auto si = cfg.speaker_ids.find(spk);
    if (si == cfg.speaker_ids.end()) invalid("missing speaker token id for " + spk);
    spk_id = si->second;
  }
  const size_t la = n == 0 ? 0 : (lookahead == 0 ? n : std::max<size_t>(1, std::min(lookahead, n)));
  const int P = 9 + (int)la;
  if ((size_t)P > max_cache_steps) invalid("prefill longer than max_cache_steps");
  const int ntr = (int)(n - la) + 1;
  std::vector<int> proj = {cfg.im_start, cfg.assistant, kNewline, cfg.tts_pad, cfg.tts_pad,
                           cfg.tts_pad, cfg.tts_pad, cfg.tts_pad, cfg.tts_bos};
  for (size_t i = 0; i < la; ++i) proj.push_back((int)ids[i]);
  for (size_t i = la; i < n; ++i) proj.push_back((int)ids[i]);
  proj.push_back(cfg.tts_eos);
  proj.push_back(cfg.tts_pad);
  for (int id : proj)
    if (id < 0 || id >= text_vocab) invalid("special text id out of range for the text vocab");
  if ((size_t)ntr > max_cache_steps + 1) invalid("too many trailing rows");
  project_text(proj, tp_c);
  const int codec_list[7] = {cfg.codec_think, cfg.codec_think_bos, li->second, cfg.codec_think_eos,
                             spk_id, cfg.codec_pad, cfg.codec_bos};
  std::vector<int> pidx(P), cids(P);
  for (int r = 0; r < 3; ++r) { pidx[r] = r; cids[r] = -1; }
  for (int i = 0; i < 6; ++i) { pidx[3 + i] = 3 + i; cids[3 + i] = codec_list[i]; }
  for (size_t i = 0; i < la; ++i) {
    pidx[9 + i] = 9 + (int)i;
    cids[9 + i] = codec_list[i + 1 == la ? 6 : 5];
  }
  if (xvec_host) h2d(xvec, xvec_host, (size_t)cfg.talker.hidden * 4);
  h2d(tp_pidx, pidx.data(), (size_t)P * 4);
  h2d(tp_cids, cids.data(), (size_t)P * 4);
  const int H = cfg.talker.hidden;
  QCK(launch_assemble_rows(tp_c, tp_pidx, codec_emb, tp_cids, xvec, P, H, tb.x, stream));
  QCK(cudaMemcpyAsync(trailing, tp_c + (size_t)P * H, (size_t)ntr * H * 4,
                      cudaMemcpyDeviceToDevice, stream));
  QCK(cudaMemcpyAsync(tts_pad, tp_c + (size_t)(P + ntr) * H, (size_t)H * 4,
                      cudaMemcpyDeviceToDevice, stream));
  *n_trailing = ntr;
  return P;
}

// ---- options (generation.rs:569-583, sampling.rs:12-26) --------------------
void Engine::validate(const qtts_generate_options& o) const {
  if (o.max_frames == 0) invalid("max_frames must be non-zero");
  if (!(o.repetition_penalty > 0.f)) invalid("repetition_penalty must be positive");
  auto check = [](const char* name, float top_p, float temp) {
    if (!(top_p > 0.f) || top_p > 1.f)
      invalid(std::string(name) + ".top_p must be in (0, 1], got " + std::to_string(top_p));
    if (!(temp > 0.f))
      invalid(std::string(name) + ".temperature must be positive, got " + std::to_string(temp));
  };
  check("talker", o.top_p, o.temperature);
  check("subtalker", o.subtalker_top_p, o.subtalker_temperature);
  if (o.rng != RNG_LCG && o.rng != RNG_PHILOX) invalid("rng must be 0 (lcg) or 1 (philox)");
}

// Starts a sequence whose prefill rows are already in the talker input:
// state reset, talker prefill and the first semantic token (generation.rs:681-693).
void Engine::begin(int P, int n_trailing, const qtts_generate_options& o) {
  if ((size_t)P + o.max_frames > max_cache_steps)
    fail(QTTS_ERR_CACHE_FULL, "requested " + std::to_string(P + o.max_frames) +
                                  " cache steps but engine was loaded for " +
                                  std::to_string(max_cache_steps) +
                                  "; call load_with_max_frames with a larger max_frames");
  SeqState s{};
  s.frames = 0;
  s.semantic = -1;
  s.talker_pos = P;
  s.prefill_len = P;
  s.n_trailing = n_trailing;
  s.rng_kind = o.rng;
  s.rng_state = o.seed ^ kSeedXor;
  s.rng_seed = o.seed;
  *st_host = s;
  QCK(cudaMemcpyAsync(st, st_host, sizeof(SeqState), cudaMemcpyHostToDevice, stream));
  QCK(cudaEventRecord(ev0, stream));
  const size_t l0 = launches;
  stack_rows(talker, tb, tkv, P, 0, nullptr);
  talker_head(ROLE_TALKER_PREFILL, tb.x + (size_t)(P - 1) * cfg.talker.hidden, talker_cfg(o),
              1.0f, nullptr, cp_prefix_target());
  QCK(cudaEventRecord(ev1, stream));
  seq_P = P;
  seq_frames = 0;
  seq_max_frames = o.max_frames;
  seq_opts = o;
  seq_ended = false;
  ++seq_id;
  sync_state();
  seq_semantic = st_host->semantic;
  QCK(cudaEventElapsedTime(&last_prefill_ms, ev0, ev1));
  last_frames_ms = 0.f;
  last_frames = 0;
  last_launches = launches - l0;
}

void Engine::sync_state() {
  QCK(cudaMemcpyAsync(st_host, st, sizeof(SeqState), cudaMemcpyDeviceToHost, stream));
  stream_sync();
  if (st_host->error)
    fail(QTTS_ERR_DEVICE_STATE, "cannot sample from logits with no finite values");
  if (tc_err) {
    int e = 0;
    QCK(cudaMemcpy(&e, tc_err, sizeof(int), cudaMemcpyDeviceToHost));
    if (e) fail(QTTS_ERR_DEVICE_STATE, "tensor-core projection pipeline timed out (stage " +
                                           std::to_string(e) + ")");
  }
  check_kv();
}

// Enqueues up to n frames (fewer if EOS stops the loop on the device) and
// returns the number of frames produced.
size_t Engine::run_frames(size_t n) {
  if (seq_ended || (size_t)seq_frames >= seq_max_frames || n == 0) return 0;
  n = std::min(n, seq_max_frames - seq_frames);
  SampleKey full{talker_cfg(seq_opts), sub_cfg(seq_opts), seq_opts.repetition_penalty, 0};
  SampleKey last = full;
  last.last = 1;
  cudaGraphExec_t gf = nullptr, gl = nullptr;
  const size_t begin = seq_frames;
  for (size_t i = 0; i < n; ++i)
    if (begin + i + 1 < seq_max_frames) gf = frame_graph(full); else gl = frame_graph(last);
  QCK(cudaEventRecord(ev1, stream));
  bool traced = false;
  for (size_t i = 0; i < n; ++i) {
    const bool is_last = begin + i + 1 >= seq_max_frames;
    const bool trace_now = trace_on && !is_last && begin + i == trace_frame;
    if (trace_now) {
      QCK(cudaMemsetAsync(step_trace, 0xff, 2 * kTraceCap * sizeof(unsigned long long), stream));
      QCK(cudaMemsetAsync(step_trace + 2 * kTraceCap, 0,
                          (6 * kTraceCap + 256) * sizeof(unsigned long long), stream));
      QCK(set_step_trace(step_trace, kTraceCap, stream));
    }
    QCK(cudaGraphLaunch(is_last ? gl : gf, stream));
    if (trace_now) {
      QCK(set_step_trace(nullptr, 0, stream));
      traced = true;
    }
    last_launches += graph_nodes[is_last ? last : full];
  }
  QCK(cudaEventRecord(ev2, stream));
  sync_state();
  if (traced) dump_step_trace();
  float ms = 0.f;
  QCK(cudaEventElapsedTime(&ms, ev1, ev2));
  last_frames_ms += ms;
  const int now = st_host->frames;
  const size_t produced = (size_t)(now - seq_frames);
  last_frames += produced;
  seq_frames = now;
  seq_semantic = st_host->semantic;
  if (st_host->halt) seq_ended = true;
  return produced;
}

void Engine::dump_step_trace() {
  std::vector<unsigned long long> t(8 * (size_t)kTraceCap);
  QCK(cudaMemcpy(t.data(), step_trace, t.size() * sizeof(unsigned long long),
                 cudaMemcpyDeviceToHost));
  unsigned long long t0 = ~0ull;
  for (size_t i = 1; i <= trace_names.size(); ++i) t0 = std::min(t0, t[i]);
  auto rel = [&](unsigned long long v) {
    return v == ~0ull || v == 0 ? -1LL : (long long)(v - t0);
  };
  trace_rows.assign(trace_names.size(), qtts_trace_launch{});
  for (size_t i = 1; i <= trace_names.size(); ++i) {
    qtts_trace_launch& r = trace_rows[i - 1];
    std::snprintf(r.name, sizeof r.name, "%s", trace_names[i - 1].c_str());
    r.entry_ns = rel(t[i]);
    r.wait_ns = rel(t[kTraceCap + i]);
    r.exit_ns = rel(t[2 * kTraceCap + i]);
    r.last_wait_ns = rel(t[3 * kTraceCap + i]);
    r.mark4_ns = rel(t[4 * kTraceCap + i]);
    r.mark5_ns = rel(t[5 * kTraceCap + i]);
    r.dur6_ns = t[6 * kTraceCap + i];
    r.dur7_ns = t[7 * kTraceCap + i];
  }
  if (step_trace_path.empty()) return;
  FILE* f = std::fopen(step_trace_path.c_str(), "w");
  if (!f) return;
  std::fprintf(f, "# id entry wait exit last_wait mark4 mark5 (ns after the first entry) "
                  "dur6 dur7 (ns after a CTA's own wait, max over CTAs) name\n");
  for (size_t i = 0; i < trace_rows.size(); ++i) {
    const qtts_trace_launch& r = trace_rows[i];
    std::fprintf(f, "%zu %lld %lld %lld %lld %lld %lld %llu %llu %s\n", i + 1,
                 (long long)r.entry_ns, (long long)r.wait_ns, (long long)r.exit_ns,
                 (long long)r.last_wait_ns, (long long)r.mark4_ns, (long long)r.mark5_ns,
                 (unsigned long long)r.dur6_ns, (unsigned long long)r.dur7_ns, r.name);
  }
  std::fclose(f);
  {
    // token selection phases of the traced frame's heads (clock64 cycles
    // between the Selector's stamps; slots 0-6 general path, 10-15 fast path)
    std::vector<long long> sv(256);
    QCK(cudaMemcpy(sv.data(), step_trace + 8 * (size_t)kTraceCap, sv.size() * sizeof(long long),
                   cudaMemcpyDeviceToHost));
    FILE* g = std::fopen((step_trace_path + ".sel").c_str(), "w");
    if (g) {
      std::fprintf(g, "# head (0 talker, 1+g CodePredictor group g): clock64 at the Selector's "
                      "stamps 0..15, relative to the first nonzero one\n");
      for (int h = 0; h < 16; ++h) {
        long long base = 0;
        for (int k = 0; k < 16; ++k)
          if (sv[16 * h + k] && (!base || sv[16 * h + k] < base)) base = sv[16 * h + k];
        std::fprintf(g, "%d", h);
        for (int k = 0; k < 16; ++k)
          std::fprintf(g, " %lld", sv[16 * h + k] ? sv[16 * h + k] - base : -1LL);
        std::fprintf(g, "\n");
      }
      std::fclose(g);
    }
  }
}

// ---- batched serving -------------------------------------------------------
void Engine::ensure_batch() {
  if (bt.cap) return;
  if (!tc.tokens) fail(QTTS_ERR_UNSUPPORTED, "batched generation needs the tensor-core projections");
  const StackCfg& T = cfg.talker;
  const StackCfg& C = cfg.cp;
  const int cap = kBatchCap;
  const size_t mcs = max_cache_steps;
  const size_t H = T.hidden;
  bt.cap = cap;
  bt.st = arena.alloc<SeqState>(cap);
  QCK(cudaMallocHost(&bt.st_host, sizeof(SeqState) * cap));
  bt.codes = arena.alloc<int>((size_t)cap * mcs * C.groups);
  bt.history = arena.alloc<int>((size_t)cap * mcs);
  bt.trailing = arena.alloc<float>((size_t)cap * (mcs + 1) * H);
  bt.cp_prefix = arena.alloc<float>((size_t)cap * 2 * H);
  bt.cp_next = arena.alloc<float>((size_t)cap * H);
  bt.emb_sum = arena.alloc<float>((size_t)cap * H);
  bt.logits = arena.alloc<float>((size_t)cap * std::max(T.vocab, C.vocab));
  bt.tb = alloc_bufs(arena, talker, cap);
  bt.cb = alloc_bufs(arena, cp, cap);
  // talker KV: cap sequences x pages each; page table row b = its pages
  bt.tkv = tkv;
  bt.pages = (int)((mcs + (1u << tkv.page_shift) - 1) >> tkv.page_shift);
  bt.tkv.pool = alloc_talker_pool(bt.pages * cap);
  {
    std::vector<int> pt((size_t)bt.pages * cap);
    for (size_t i = 0; i < pt.size(); ++i) pt[i] = (int)i;
    int* d = arena.alloc<int>(pt.size());
    h2d(d, pt.data(), pt.size() * 4);
    bt.tkv.page_table = d;
  }
  // CodePredictor KV: one page (all its positions) per sequence
  bt.ckv = ckv;
  bt.ckv.pool = arena.alloc<__nv_bfloat16>((size_t)(ckv.page_stride * cap));
  {
    std::vector<int> pt(cap);
    for (int i = 0; i < cap; ++i) pt[i] = i;
    int* d = arena.alloc<int>(cap);
    h2d(d, pt.data(), (size_t)cap * 4);
    bt.ckv.page_table = d;
  }
  // 16-row token tiles with a split-K workspace
  bt.rms = arena.alloc<float>(cap);
  bt.plan.tokens = 16;
  bt.plan.sm_count = tc.sm_count;
  bt.plan.max_splits = 16;
  bt.plan.ws_floats = tc_workspace_floats(16, tc.sm_count);
  bt.plan.ws = arena.alloc<float>(bt.plan.ws_floats);
  bt.plan.tickets = arena.alloc<unsigned>(4096);
  for (auto& ev : bt.ev) QCK(cudaEventCreate(&ev));
}

void Engine::blinear(const __nv_bfloat16* W, const float* x, int ldx, const float* gamma,
                     float eps, float* y, int ldy, const float* resid, int ldr, const float* bias,
                     int M, int N, int K, Epilogue epi, float* rms_out) {
  LinearArgs a{W, x, ldx, gamma, eps, y, ldy, resid, ldr, bias, M, N, K, nullptr};
  if (!tc_supported(a, epi, bt.plan))
    fail(QTTS_ERR_UNSUPPORTED, "projection shape unsupported by the batched tensor-core path");
  QCK(launch_linear_tc(a, epi, bt.plan, rms_out, tc_err, stream));
  launches += 1;
}

// One position through all layers for nb sequences (rows of B.x).
void Engine::batch_stack_step(DevStack& S, StackBufs& B, const KvView& kv, int pt_stride,
                              const int* pos_ptr, int pos_const, int nb, bool qkv0_given) {
  const StackCfg& c = S.c;
  const float scale = 1.0f / std::sqrt((float)c.head_dim);
  for (int l = 0; l < c.layers; ++l) {
    if (!(l == 0 && qkv0_given))  // else: rows of the precomputed table, written by the heads
      blinear(S.wqkv[l], B.x, c.hidden, S.in_g[l], c.eps, B.qkv, S.qkv_w, nullptr, 0, nullptr,
              nb, S.qkv_w, c.hidden, EPI_STORE);
    constexpr int kStride = (int)(sizeof(SeqState) / sizeof(int));
    if (&S == &talker && kv_form()) {
      kv_attention(S, B, kv_args(kv, nb, pt_stride, pos_ptr, kStride, pos_const),
                   KvRows{nullptr, nullptr, nb, nb, 1, 0, 0}, l, &bt.st[0].halt, kStride);
    } else {
    AttnDecodeArgs da{};
    da.qkv = B.qkv;
    da.q_gamma = S.q_g[l];
    da.k_gamma = S.k_g[l];
    da.eps = c.eps;
    da.rope_cos = S.rope_cos;
    da.rope_sin = S.rope_sin;
    da.kv = kv;
    da.layer = l;
    da.pos_ptr = pos_ptr;
    da.pos_const = pos_const;
    da.q_heads = c.q_heads;
    da.scale = scale;
    da.out = B.attn;
    da.halt = &bt.st[0].halt;
    da.qkv_ld = S.qkv_w;
    da.out_ld = S.q_out;
    da.pos_stride = kStride;
    da.halt_stride = kStride;
    da.pt_stride = pt_stride;
    da.batch = nb;
    QCK(launch_attn_decode(da, stream));
    ++launches;
    }
    blinear(S.wo[l], B.attn, S.q_out, nullptr, 0.f, B.h1, c.hidden, B.x, c.hidden, nullptr, nb,
            c.hidden, S.q_out, EPI_RESID);
    blinear(S.wgu[l], B.h1, c.hidden, S.post_g[l], c.eps, B.act, c.intermediate, nullptr, 0,
            nullptr, nb, c.intermediate, c.hidden, EPI_SWIGLU);
    blinear(S.wdown[l], B.act, c.intermediate, nullptr, 0.f, B.x, c.hidden, B.h1, c.hidden,
            nullptr, nb, c.hidden, c.intermediate, EPI_RESID);
  }
}

void Engine::batch_head(int role, int group, const float* x, const SampleCfg& c, float penalty,
                        int nb) {
  const StackCfg& T = cfg.talker;
  const StackCfg& C = cfg.cp;
  const bool talker_role = role != ROLE_CP_GROUP;
  const StackCfg& S = talker_role ? T : C;
  const __nv_bfloat16* W = talker_role ? head : cp_heads + (size_t)group * C.vocab * C.hidden;
  const float* gamma = talker_role ? norm_g : cp_norm_g;
  blinear(W, x, S.hidden, gamma, S.eps, bt.logits, S.vocab, nullptr, 0, nullptr, nb, S.vocab,
          S.hidden, EPI_STORE, bt.rms);
  BatchHeadArgs bh{};
  HeadArgs& a = bh.h;
  a.role = role;
  a.cfg = c;
  a.st = bt.st;
  a.penalty = talker_role ? penalty : 1.0f;
  a.history = bt.history;
  a.history_out = bt.history;
  a.eos_token = cfg.codec_eos;
  a.suppress = talker_role ? 1 : 0;
  a.talker_codec_emb = codec_emb;
  a.H = T.hidden;
  a.groups = C.groups;
  a.codes = bt.codes;
  a.lin = LinearArgs{W, x, S.hidden, gamma, S.eps, bt.logits, S.vocab, nullptr, 0, nullptr, 1,
                     S.vocab, S.hidden, nullptr};
  a.frames_cap = (int)max_cache_steps;
  a.talker_vocab = T.vocab;
  if (talker_role) {
    a.cp_prefix = bt.cp_prefix;
  } else {
    a.group = group;
    a.last_group = C.groups - 2;
    a.cp_emb = cp_embs + (size_t)group * C.vocab * T.hidden;
    a.cp_next = has_proj() ? bt.cp_next : bt.cb.x;
    a.emb_sum = bt.emb_sum;
    a.step_in = bt.tb.x;
    a.trailing = bt.trailing;
    a.tts_pad = tts_pad;
  }
  bh.logits = bt.logits;
  bh.logits_ld = S.vocab;
  bh.rms = bt.rms;
  bh.hist_stride = (long long)max_cache_steps;
  bh.codes_stride = (long long)max_cache_steps * C.groups;
  bh.next_stride = has_proj() ? T.hidden : C.hidden;
  bh.step_stride = T.hidden;
  bh.trail_stride = (long long)(max_cache_steps + 1) * T.hidden;
  if (!talker_role && cp_qkv0 && group < C.groups - 2) {
    a.qkv_table = cp_qkv0 + (size_t)group * C.vocab * cp.qkv_w;
    a.qkv_out = bt.cb.qkv;
    a.qkv_w = cp.qkv_w;
    bh.qkv_stride = cp.qkv_w;
    if (cp_x0) {
      a.x_table = cp_x0 + (size_t)group * C.vocab * C.hidden;
      a.x_out = bt.cb.x;
      a.x_w = C.hidden;
      bh.x_stride = C.hidden;
    }
  }
  QCK(launch_select_batch(bh, nb, stream));
  ++launches;
}

// One frame for nb sequences: CodePredictor positions 0 and 1 (its 2-row
// prefill, as two decode steps), head 0, groups 1..14, then unless last the
// talker step and its token (same order as enqueue_frame).
void Engine::enqueue_batch_frame(const SampleKey& k, int nb, const KvView& view) {
  const StackCfg& T = cfg.talker;
  const StackCfg& C = cfg.cp;
  const size_t H = T.hidden;
  for (int j = 0; j < 2; ++j) {
    if (has_proj()) {
      blinear(proj_w, bt.cp_prefix + j * H, 2 * (int)H, nullptr, 0.f, bt.cb.x, C.hidden, nullptr,
              0, proj_b, nb, C.hidden, (int)H, EPI_BIAS);
    } else {
      QCK(cudaMemcpy2DAsync(bt.cb.x, C.hidden * sizeof(float), bt.cp_prefix + j * H,
                            2 * H * sizeof(float), H * sizeof(float), nb,
                            cudaMemcpyDeviceToDevice, stream));
    }
    batch_stack_step(cp, bt.cb, bt.ckv, 1, nullptr, j, nb);
  }
  batch_head(ROLE_CP_GROUP, 0, bt.cb.x, k.s, 1.0f, nb);
  for (int g = 1; g < C.groups - 1; ++g) {
    if (has_proj() && !cp_x0)
      blinear(proj_w, bt.cp_next, (int)H, nullptr, 0.f, bt.cb.x, C.hidden, nullptr, 0, proj_b, nb,
              C.hidden, (int)H, EPI_BIAS);
    batch_stack_step(cp, bt.cb, bt.ckv, 1, nullptr, g + 1, nb, cp_qkv0 != nullptr);
    batch_head(ROLE_CP_GROUP, g, bt.cb.x, k.s, 1.0f, nb);
  }
  if (!k.last) {
    batch_stack_step(talker, bt.tb, view, bt.pages, &bt.st[0].talker_pos, 0, nb);
    batch_head(ROLE_TALKER_STEP, 0, bt.tb.x, k.t, k.penalty, nb);
  }
}

cudaGraphExec_t Engine::batch_graph(const SampleKey& k, int nb, const KvView& view, bool takes) {
  auto key = std::make_pair(k, takes ? -nb : nb);
  auto it = batch_graphs.find(key);
  if (it != batch_graphs.end()) return it->second;
  cudaGraph_t g = nullptr;
  const size_t before = launches;
  QCK(cudaStreamBeginCapture(stream, cudaStreamCaptureModeThreadLocal));
  try {
    enqueue_batch_frame(k, nb, view);
  } catch (...) {
    cudaStreamEndCapture(stream, &g);
    if (g) cudaGraphDestroy(g);
    launches = before;
    throw;
  }
  QCK(cudaStreamEndCapture(stream, &g));
  batch_nodes[key] = launches - before;
  launches = before;
  cudaGraphExec_t exec = nullptr;
  cudaError_t e = cudaGraphInstantiate(&exec, g, 0);
  cudaGraphDestroy(g);
  QCK(e);
  batch_graphs[key] = exec;
  return exec;
}

// The state that a prefill left (sequence, CodePredictor prefix, trailing rows)
// into batch slot b.
void Engine::store_slot(int b, int ntr) {
  const size_t H = cfg.talker.hidden;
  QCK(cudaMemcpyAsync(bt.st + b, st, sizeof(SeqState), cudaMemcpyDeviceToDevice, stream));
  QCK(cudaMemcpyAsync(bt.cp_prefix + (size_t)b * 2 * H, cp_prefix_target(),
                      2 * H * sizeof(float), cudaMemcpyDeviceToDevice, stream));
  QCK(cudaMemcpyAsync(bt.trailing + (size_t)b * (max_cache_steps + 1) * H, trailing,
                      (size_t)ntr * H * sizeof(float), cudaMemcpyDeviceToDevice, stream));
}

void Engine::generate_batch(const std::vector<std::vector<uint32_t>>& ids,
                            const std::vector<qtts_generate_options>& opts, int32_t* codes_out,
                            size_t cap_per_request, size_t* frames_out, int32_t* ended_out) {
  const int nb = (int)ids.size();
  if (nb < 1 || nb > kBatchCap)
    invalid("batch size must be in [1, " + std::to_string(kBatchCap) + "]");
  const qtts_generate_options& o0 = opts[0];
  for (const auto& o : opts) {
    validate(o);
    if (o.max_frames != o0.max_frames || o.do_sample != o0.do_sample || o.top_k != o0.top_k ||
        o.top_p != o0.top_p || o.temperature != o0.temperature ||
        o.repetition_penalty != o0.repetition_penalty ||
        o.subtalker_dosample != o0.subtalker_dosample ||
        o.subtalker_top_k != o0.subtalker_top_k || o.subtalker_top_p != o0.subtalker_top_p ||
        o.subtalker_temperature != o0.subtalker_temperature || o.rng != o0.rng)
      invalid("batched requests must share every option except seed, speaker and language");
  }
  const size_t G = cfg.cp.groups;
  if (cap_per_request < (size_t)o0.max_frames * G) invalid("codes_out capacity too small");
  ensure_batch();
  // prefill each request into its slot (the single-sequence path on the slot's KV view)
  const KvView saved = tkv;
  QCK(cudaEventRecord(bt.ev[0], stream));
  try {
    for (int b = 0; b < nb; ++b) {
      int ntr = 0;
      const int P = prepare(ids[b].data(), ids[b].size(), 0, opts[b].speaker, opts[b].language,
                            nullptr, &ntr);
      tkv = bt.tkv;
      tkv.page_table = bt.tkv.page_table + (size_t)b * bt.pages;
      begin(P, ntr, opts[b]);
      tkv = saved;
      store_slot(b, ntr);
    }
  } catch (const QttsError& err) {
    tkv = saved;
    if (!crumbs_host) throw;
    fail(err.code, std::string(err.what()) + " [prefill; last kernel entered " +
                       std::to_string(crumbs_host[0]) + ", last gemm left " +
                       std::to_string(crumbs_host[1]) + "]");
  } catch (...) {
    tkv = saved;
    throw;
  }
  run_batch(nb, o0, bt.tkv, false, codes_out, cap_per_request, frames_out, ended_out);
}

// Frames of nb prefilled slots until every one has ended or has max_frames.
void Engine::run_batch(int nb, const qtts_generate_options& o0, const KvView& view, bool takes,
                       int32_t* codes_out, size_t cap_per_request, size_t* frames_out,
                       int32_t* ended_out) {
  const size_t G = cfg.cp.groups;
  SampleKey full{talker_cfg(o0), sub_cfg(o0), o0.repetition_penalty, 0};
  SampleKey last = full;
  last.last = 1;
  const size_t max_frames = o0.max_frames;
  // QTTS_BATCH_EAGER=1: enqueue the kernels directly instead of replaying a
  // graph (debugging aid: launch errors surface at the launch that caused them)
  const char* eg = std::getenv("QTTS_BATCH_EAGER");
  const bool eager = eg && eg[0] == '1';
  cudaGraphExec_t gf = !eager && max_frames > 1 ? batch_graph(full, nb, view, takes) : nullptr;
  cudaGraphExec_t gl = eager ? nullptr : batch_graph(last, nb, view, takes);
  size_t done = 0;
  last_launches = 0;
  QCK(cudaEventRecord(bt.ev[1], stream));
  try {
  while (done < max_frames) {
    const size_t burst = std::min<size_t>(16, max_frames - done);
    for (size_t i = 0; i < burst; ++i) {
      const bool is_last = done + i + 1 >= max_frames;
      if (eager) {
        enqueue_batch_frame(is_last ? last : full, nb, view);
        QCK(cudaStreamSynchronize(stream));
        continue;
      }
      QCK(cudaGraphLaunch(is_last ? gl : gf, stream));
      last_launches += batch_nodes[std::make_pair(is_last ? last : full, takes ? -nb : nb)];
    }
    done += burst;
    QCK(cudaMemcpyAsync(bt.st_host, bt.st, sizeof(SeqState) * nb, cudaMemcpyDeviceToHost,
                        stream));
    QCK(cudaStreamSynchronize(stream));
    bool all_halted = true;
    for (int b = 0; b < nb; ++b) all_halted = all_halted && bt.st_host[b].halt;
    if (all_halted) break;
  }
  } catch (const QttsError& err) {
    if (!crumbs_host) throw;
    std::string st_dump;
    for (int b = 0; b < nb; ++b)
      st_dump += " [" + std::to_string(b) + ": f" + std::to_string(bt.st_host[b].frames) + " s" +
                 std::to_string(bt.st_host[b].semantic) + " p" +
                 std::to_string(bt.st_host[b].talker_pos) + " h" +
                 std::to_string(bt.st_host[b].halt) + "]";
    fail(err.code, std::string(err.what()) + " [last kernel entered " +
                       std::to_string(crumbs_host[0]) + ", last gemm left " +
                       std::to_string(crumbs_host[1]) + ", check " +
                       std::to_string(crumbs_host[2]) + " v " + std::to_string(crumbs_host[3]) +
                       " " + std::to_string(crumbs_host[4]) + " seq " +
                       std::to_string(crumbs_host[5]) + ", frames done " + std::to_string(done) +
                       "; last synced state:" + st_dump + "]");
  }
  QCK(cudaEventRecord(bt.ev[2], stream));
  QCK(cudaStreamSynchronize(stream));
  QCK(cudaEventElapsedTime(&last_prefill_ms, bt.ev[0], bt.ev[1]));
  QCK(cudaEventElapsedTime(&last_frames_ms, bt.ev[1], bt.ev[2]));
  int tc_e = 0;
  QCK(cudaMemcpy(&tc_e, tc_err, sizeof(int), cudaMemcpyDeviceToHost));
  if (tc_e) fail(QTTS_ERR_DEVICE_STATE, "tensor-core projection pipeline timed out");
  check_kv();
  last_frames = 0;
  for (int b = 0; b < nb; ++b) {
    const SeqState& s = bt.st_host[b];
    if (s.error == 1) fail(QTTS_ERR_DEVICE_STATE, "cannot sample from logits with no finite values");
    if (s.error)
      fail(QTTS_ERR_DEVICE_STATE,
           "batched head found an out-of-range sequence state (code " + std::to_string(s.error) +
               (crumbs_host ? ", check " + std::to_string(crumbs_host[2]) + " v " +
                                  std::to_string(crumbs_host[3]) + " " +
                                  std::to_string(crumbs_host[4]) + " seq " +
                                  std::to_string(crumbs_host[5])
                            : std::string()) +
               ")");
    const size_t f = (size_t)s.frames;
    QCK(cudaMemcpy(codes_out + (size_t)b * cap_per_request, bt.codes + (size_t)b * max_cache_steps * G,
                   f * G * sizeof(int32_t), cudaMemcpyDeviceToHost));
    if (frames_out) frames_out[b] = f;
    if (ended_out) ended_out[b] = s.halt ? 1 : 0;
    last_frames += f;
  }
}

// ---- takes: one prompt, several seeds ---------------------------------------
void Engine::ensure_takes() {
  if (bt.takes.table) return;
  KvArgs& c = bt.takes;
  c.g = KvGeom{bt.pages * bt.cap, bt.cap, bt.pages, cfg.talker.layers, cfg.talker.kv_heads,
               bt.tkv.page_shift, cache.kv_bits};
  c.pool = reinterpret_cast<unsigned char*>(bt.tkv.pool);
  c.lengths = arena.alloc<int>(bt.cap);
  c.len_stride = 1;
  c.refs = arena.alloc<int>(c.g.pages);
  c.work = arena.alloc<int>(kv_work_ints(c.g));
  c.table = arena.alloc<int>((size_t)bt.pages * bt.cap);
}

// The prompt is prefilled once into take 0; the others fork its pages (full ones
// are shared, the last one is copied) and draw their first token from the same
// logits with their own seeds. Frames then run as a batch's do.
void Engine::generate_takes(const uint32_t* ids, size_t n, const qtts_generate_options& o,
                            const std::vector<uint64_t>& seeds, int32_t* codes_out,
                            size_t cap_per_take, size_t* frames_out, int32_t* ended_out) {
  const int nb = (int)seeds.size();
  if (nb < 1 || nb > kBatchCap) invalid("takes must be in [1, " + std::to_string(kBatchCap) + "]");
  validate(o);
  if (cap_per_take < (size_t)o.max_frames * cfg.cp.groups) invalid("codes_out capacity too small");
  ensure_batch();
  ensure_takes();
  int ntr = 0;
  QCK(cudaEventRecord(bt.ev[0], stream));
  const int P = prepare(ids, n, 0, o.speaker, o.language, nullptr, &ntr);
  if ((size_t)P + o.max_frames > max_cache_steps)
    fail(QTTS_ERR_CACHE_FULL, "requested " + std::to_string(P + o.max_frames) +
                                  " cache steps but engine was loaded for " +
                                  std::to_string(max_cache_steps));
  KvArgs& c = bt.takes;
  QCK(cudaMemsetAsync(c.table, 0xff, (size_t)c.g.max_pages * c.g.seqs * sizeof(int), stream));
  QCK(cudaMemsetAsync(c.lengths, 0, c.g.seqs * sizeof(int), stream));
  QCK(cudaMemsetAsync(c.refs, 0, (size_t)c.g.pages * sizeof(int), stream));
  KvList list;
  list.n = 1;
  list.a[0] = 0;
  list.b[0] = P;
  QCK(launch_kv_resize(c, list, stream));
  KvView view = bt.tkv;
  view.page_table = c.table;
  const KvView saved = tkv;
  qtts_generate_options first = o;
  first.seed = seeds[0];
  tkv = view;
  try {
    begin(P, ntr, first);
  } catch (...) {
    tkv = saved;
    throw;
  }
  tkv = saved;
  store_slot(0, ntr);
  for (int b = 1; b < nb; ++b) {
    SeqState s{};
    s.semantic = -1;
    s.talker_pos = P;
    s.prefill_len = P;
    s.n_trailing = ntr;
    s.rng_kind = o.rng;
    s.rng_state = seeds[b] ^ kSeedXor;
    s.rng_seed = seeds[b];
    h2d(st, &s, sizeof s);
    talker_head(ROLE_TALKER_PREFILL, tb.x + (size_t)(P - 1) * cfg.talker.hidden, talker_cfg(o), 1.0f,
                nullptr, cp_prefix_target());
    store_slot(b, ntr);
  }
  list.n = nb - 1;
  for (int b = 1; b < nb; ++b) {
    list.a[b - 1] = 0;
    list.b[b - 1] = b;
  }
  QCK(launch_kv_fork(c, list, stream));
  list.n = nb;
  for (int b = 0; b < nb; ++b) {
    list.a[b] = b;
    list.b[b] = P + (int)o.max_frames;
  }
  QCK(launch_kv_resize(c, list, stream));
  int e = 0;
  QCK(cudaMemcpyAsync(&e, c.work, sizeof e, cudaMemcpyDeviceToHost, stream));
  stream_sync();
  if (e) {
    QCK(cudaMemset(c.work, 0, sizeof e));
    fail(QTTS_ERR_DEVICE_STATE, "page management reported status " + std::to_string(e));
  }
  run_batch(nb, o, view, true, codes_out, cap_per_take, frames_out, ended_out);
  // no stream of an earlier generation may continue: take 0 ended this one
  seq_ended = true;
}

void Engine::read_codes(size_t from, size_t to, int32_t* out) {
  if (to <= from) return;
  const size_t g = cfg.cp.groups;
  QCK(cudaMemcpy(out, codes + from * g, (to - from) * g * 4, cudaMemcpyDeviceToHost));
}

// ---------------------------------------------------------------------------
struct Stream {
  Engine* e;
  uint64_t id;
  size_t max_frames;
  std::vector<int32_t> codes;
};

// PollingTextStream (generation.rs:1086-1451) on token ids.
struct TextStream {
  Engine* e;
  qtts_generate_options opts;
  qtts_text_stream_options topts;
  std::deque<uint32_t> queued;
  bool text_finished = false, eos_pending = false, eos_consumed = false;
  bool started = false, finished = false;
  uint64_t id = 0;
  std::vector<int32_t> codes;
};

}  // namespace
}  // namespace qtts

using qtts::Engine;
using qtts::guard;
using qtts::need;
using qtts::QttsError;

struct qtts_engine {
  std::unique_ptr<Engine> e;
};
struct qtts_stream {
  qtts::Stream s;
};
struct qtts_text_stream {
  qtts::TextStream s;
};
struct qtts_codec_stream {
  qtts::Engine* e;
  std::unique_ptr<qtts::Codec::StreamState> st;
};

namespace {

Engine& engine_of(qtts_engine* e) {
  need(e, "engine");
  QCK(cudaSetDevice(e->e->device));
  return *e->e;
}

void finish_generation(Engine& e, int32_t* codes_out, size_t cap, size_t* frames_out,
                       int32_t* ended) {
  e.run_frames(e.seq_max_frames);
  const size_t g = e.cfg.cp.groups;
  if (cap < (size_t)e.seq_frames * g) qtts::invalid("codes_out capacity too small");
  e.read_codes(0, e.seq_frames, codes_out);
  if (frames_out) *frames_out = e.seq_frames;
  if (ended) *ended = e.seq_ended ? 1 : 0;
}

int32_t load_engine(const char* dir, int32_t device, const qtts_cache_options& cache,
                    qtts_engine** out) {
  return guard([&] {
    need(dir, "model_dir");
    need(out, "out");
    *out = nullptr;
    auto h = std::make_unique<qtts_engine>();
    h->e = std::make_unique<Engine>(dir, device, cache);
    *out = h.release();
  });
}

// Host side of next_trailing_buffer (generation.rs:1360-1388): the text id of
// the next trailing row, or -1 when no row is ready yet.
long long next_trailing_id(qtts::TextStream& s) {
  const Engine& e = *s.e;
  if (!s.text_finished && s.queued.size() < s.topts.min_resume_tokens) return -1;
  if (!s.queued.empty()) {
    const uint32_t t = s.queued.front();
    s.queued.pop_front();
    return t;
  }
  if (s.eos_pending) {
    s.eos_pending = false;
    s.eos_consumed = true;
    return e.cfg.tts_eos;
  }
  if (s.text_finished || s.eos_consumed) return e.cfg.tts_pad;
  return -1;
}

}  // namespace

extern "C" {

const char* qtts_last_error(void) { return qtts::last_error().c_str(); }
int32_t qtts_abi_version(void) { return 2; }

void qtts_generate_options_default(qtts_generate_options* o) {
  if (!o) return;
  *o = qtts_generate_options{};
  o->speaker = "ryan";
  o->language = "english";
  o->max_frames = 240;
  o->decode_audio = 0;
  o->do_sample = 1;
  o->top_k = 50;
  o->top_p = 1.0f;
  o->temperature = 0.9f;
  o->repetition_penalty = 1.05f;
  o->subtalker_dosample = 1;
  o->subtalker_top_k = 50;
  o->subtalker_top_p = 1.0f;
  o->subtalker_temperature = 0.9f;
  o->seed = 0;
  o->rng = 0;
}

void qtts_stream_options_default(qtts_stream_options* o) {
  if (!o) return;
  o->text_lookahead_tokens = 8;
  o->left_context_frames = 25;
}

void qtts_text_stream_options_default(qtts_text_stream_options* o) {
  if (!o) return;
  o->min_start_tokens = 8;
  o->min_resume_tokens = 1;
  o->flush_on_punctuation = 1;
  o->left_context_frames = 25;
}

int32_t qtts_engine_load(const char* dir, int32_t device, qtts_engine** out) {
  return load_engine(dir, device, {512, 16, 0, 0}, out);
}

int32_t qtts_engine_load_with_max_frames(const char* dir, int32_t device, size_t max_frames,
                                         qtts_engine** out) {
  if (max_frames == 0) {
    qtts::last_error() = "max_frames must be non-zero";
    return QTTS_ERR_INVALID_INPUT;
  }
  return load_engine(dir, device, {256 + max_frames, 16, 0, 0}, out);
}

int32_t qtts_engine_load_with_options(const char* dir, int32_t device, size_t mcs,
                                      qtts_engine** out) {
  return load_engine(dir, device, {mcs, 16, 0, 0}, out);
}

void qtts_cache_options_default(qtts_cache_options* o) {
  if (!o) return;
  *o = qtts_cache_options{512, 16, 0, 0};
}

int32_t qtts_engine_load_with_cache(const char* dir, int32_t device,
                                    const qtts_cache_options* cache, qtts_engine** out) {
  if (!cache) {
    qtts::last_error() = "cache must not be null";
    return QTTS_ERR_INVALID_INPUT;
  }
  return load_engine(dir, device, *cache, out);
}

void qtts_engine_destroy(qtts_engine* e) { delete e; }

int32_t qtts_engine_get_info(const qtts_engine* h, qtts_engine_info* out) {
  return guard([&] {
    need(h, "engine");
    need(out, "out");
    const Engine& e = *h->e;
    out->hidden = e.cfg.talker.hidden;
    out->vocab = e.cfg.talker.vocab;
    out->cp_hidden = e.cfg.cp.hidden;
    out->cp_vocab = e.cfg.cp.vocab;
    out->num_code_groups = e.cfg.cp.groups;
    out->talker_layers = e.cfg.talker.layers;
    out->cp_layers = e.cfg.cp.layers;
    out->codec_eos = e.cfg.codec_eos;
    out->max_cache_steps = e.max_cache_steps;
    out->device_bytes = e.arena.bytes() + (e.codec ? e.codec->device_bytes() : 0);
    out->reserved[0] = out->reserved[1] = 0;
    out->has_codec = e.codec ? 1 : 0;
    out->samples_per_frame = qtts::Codec::samples_per_frame();
  });
}

int32_t qtts_decode_codes(qtts_engine* h, const int32_t* codes, size_t n_codes, float* samples,
                          size_t cap, size_t* n_samples) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(n_samples, "n_samples");
    if (n_codes) {
      need(codes, "codes");
      need(samples, "samples");
    }
    *n_samples = e.decode_codes(codes, n_codes, samples, cap);
  });
}

int32_t qtts_codec_stream_open(qtts_engine* h, size_t max_frames, qtts_codec_stream** out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(out, "out");
    *out = nullptr;
    if (!e.codec) qtts::fail(QTTS_ERR_UNSUPPORTED, "no codec: speech_tokenizer/model.safetensors not found");
    if (max_frames == 0 || max_frames > (size_t)INT32_MAX / qtts::Codec::samples_per_frame())
      qtts::invalid("max_frames must be in [1, " +
              std::to_string(INT32_MAX / qtts::Codec::samples_per_frame()) + "]");
    auto s = std::make_unique<qtts_codec_stream>();
    s->e = &e;
    s->st = e.codec->open_stream((int)max_frames);
    *out = s.release();
  });
}

int32_t qtts_codec_stream_decode(qtts_codec_stream* s, const int32_t* codes, size_t n_codes,
                                 float* samples, size_t cap, size_t* n_samples) {
  return guard([&] {
    need(s, "stream");
    need(n_samples, "n_samples");
    if (n_codes) {
      need(codes, "codes");
      need(samples, "samples");
    }
    Engine& e = *s->e;
    QCK(cudaSetDevice(e.device));
    if (n_codes % qtts::Codec::kGroups == 0 &&
        (size_t)s->st->frames + n_codes / qtts::Codec::kGroups > (size_t)s->st->cap)
      qtts::invalid("codec stream holds " + std::to_string(s->st->cap) + " frames; " +
              std::to_string(s->st->frames) + " decoded");
    *n_samples = e.decode_codes(codes, n_codes, samples, cap, s->st.get());
  });
}

void qtts_codec_stream_destroy(qtts_codec_stream* s) {
  if (!s) return;
  cudaSetDevice(s->e->device);
  delete s;
}

int32_t qtts_last_decode_timing(const qtts_engine* h, float* ms, size_t* launches) {
  return guard([&] {
    need(h, "engine");
    const Engine& e = *h->e;
    if (ms) *ms = e.last_decode_ms;
    if (launches) *launches = e.codec ? e.codec->launches : 0;
  });
}

int32_t qtts_generate_codes_from_ids(qtts_engine* h, const uint32_t* ids, size_t n,
                                     const qtts_generate_options* o, int32_t* codes_out,
                                     size_t cap, size_t* frames_out, int32_t* ended) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(o, "options");
    need(codes_out, "codes_out");
    if (n) need(ids, "content_ids");
    e.validate(*o);
    int ntr = 0;
    const int P = e.prepare(ids, n, 0, o->speaker, o->language, nullptr, &ntr);
    e.begin(P, ntr, *o);
    finish_generation(e, codes_out, cap, frames_out, ended);
  });
}

int32_t qtts_generate_codes_batch_from_ids(qtts_engine* h, const uint32_t* ids,
                                           const size_t* lengths, size_t batch,
                                           const qtts_generate_options* opts, int32_t* codes_out,
                                           size_t cap_per_request, size_t* frames_out,
                                           int32_t* ended_out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(lengths, "lengths");
    need(opts, "options");
    need(codes_out, "codes_out");
    if (batch == 0) qtts::invalid("batch must be non-zero");
    std::vector<std::vector<uint32_t>> reqs(batch);
    size_t off = 0;
    for (size_t b = 0; b < batch; ++b) {
      if (lengths[b]) need(ids, "content_ids");
      reqs[b].assign(ids + off, ids + off + lengths[b]);
      off += lengths[b];
    }
    std::vector<qtts_generate_options> o(opts, opts + batch);
    e.generate_batch(reqs, o, codes_out, cap_per_request, frames_out, ended_out);
  });
}

int32_t qtts_generate_codes_takes_from_ids(qtts_engine* h, const uint32_t* ids, size_t n,
                                           const qtts_generate_options* o, const uint64_t* seeds,
                                           size_t takes, int32_t* codes_out, size_t cap_per_take,
                                           size_t* frames_out, int32_t* ended_out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(o, "options");
    need(seeds, "seeds");
    need(codes_out, "codes_out");
    if (n) need(ids, "content_ids");
    if (takes == 0) qtts::invalid("takes must be non-zero");
    if (takes > 4096) qtts::invalid("too many takes");
    e.generate_takes(ids, n, *o, std::vector<uint64_t>(seeds, seeds + takes), codes_out,
                     cap_per_take, frames_out, ended_out);
  });
}

int32_t qtts_generate_voice_clone_codes_from_ids(qtts_engine* h, const uint32_t* ids, size_t n,
                                                 const float* spk, const qtts_generate_options* o,
                                                 int32_t* codes_out, size_t cap,
                                                 size_t* frames_out, int32_t* ended) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(o, "options");
    need(spk, "speaker_embedding");
    need(codes_out, "codes_out");
    if (n) need(ids, "content_ids");
    e.validate(*o);
    int ntr = 0;
    const int P = e.prepare(ids, n, 0, nullptr, o->language, spk, &ntr);
    e.begin(P, ntr, *o);
    finish_generation(e, codes_out, cap, frames_out, ended);
  });
}

int32_t qtts_generate_codes_from_rows(qtts_engine* h, const float* prefill, size_t P,
                                      const float* trailing, size_t T, const float* pad,
                                      const qtts_generate_options* o, int32_t* codes_out,
                                      size_t cap, size_t* frames_out, int32_t* ended) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(o, "options");
    need(prefill, "prefill");
    need(pad, "tts_pad");
    need(codes_out, "codes_out");
    if (T) need(trailing, "trailing");
    e.validate(*o);
    if (P == 0) qtts::invalid("prefill steps must be non-zero");
    if (P > e.max_cache_steps) qtts::invalid("prefill longer than max_cache_steps");
    const size_t H = e.cfg.talker.hidden;
    const size_t Tn = std::min(T, e.max_cache_steps + 1);
    e.h2d(e.tb.x, prefill, P * H * 4);
    if (Tn) e.h2d(e.trailing, trailing, Tn * H * 4);
    e.h2d(e.tts_pad, pad, H * 4);
    e.begin((int)P, (int)Tn, *o);
    finish_generation(e, codes_out, cap, frames_out, ended);
  });
}

int32_t qtts_prepare_inputs_from_ids(qtts_engine* h, const uint32_t* ids, size_t n,
                                     size_t lookahead, const char* speaker, const char* language,
                                     float* prefill_out, size_t* prefill_steps,
                                     float* trailing_out, size_t* trailing_steps,
                                     float* pad_out) {
  return guard([&] {
    Engine& e = engine_of(h);
    if (n) need(ids, "content_ids");
    int ntr = 0;
    const int P = e.prepare(ids, n, lookahead, speaker, language, nullptr, &ntr);
    const size_t H = e.cfg.talker.hidden;
    QCK(cudaStreamSynchronize(e.stream));
    if (prefill_out) QCK(cudaMemcpy(prefill_out, e.tb.x, P * H * 4, cudaMemcpyDeviceToHost));
    if (trailing_out)
      QCK(cudaMemcpy(trailing_out, e.trailing, ntr * H * 4, cudaMemcpyDeviceToHost));
    if (pad_out) QCK(cudaMemcpy(pad_out, e.tts_pad, H * 4, cudaMemcpyDeviceToHost));
    if (prefill_steps) *prefill_steps = P;
    if (trailing_steps) *trailing_steps = ntr;
  });
}

int32_t qtts_stream_start_from_ids(qtts_engine* h, const uint32_t* ids, size_t n,
                                   const qtts_generate_options* o,
                                   const qtts_stream_options* so, qtts_stream** out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(o, "options");
    need(out, "out");
    *out = nullptr;
    if (n) need(ids, "content_ids");
    e.validate(*o);
    qtts_stream_options sopt;
    qtts_stream_options_default(&sopt);
    if (so) sopt = *so;
    if (sopt.text_lookahead_tokens == 0) qtts::invalid("text_lookahead_tokens must be non-zero");
    int ntr = 0;
    const int P = e.prepare(ids, n, sopt.text_lookahead_tokens, o->speaker, o->language, nullptr,
                            &ntr);
    e.begin(P, ntr, *o);
    auto s = std::make_unique<qtts_stream>();
    s->s.e = &e;
    s->s.id = e.seq_id;
    s->s.max_frames = o->max_frames;
    *out = s.release();
  });
}

int32_t qtts_stream_next_codes_chunk(qtts_stream* h, size_t max_chunk, int32_t* codes_out,
                                     size_t cap, qtts_codes_chunk* chunk) {
  return guard([&] {
    need(h, "stream");
    need(chunk, "chunk");
    Engine& e = *h->s.e;
    QCK(cudaSetDevice(e.device));
    if (max_chunk == 0) qtts::invalid("max_chunk_frames must be non-zero");
    if (h->s.id != e.seq_id) qtts::invalid("stream was superseded by a newer generation on this engine");
    const size_t before = e.seq_frames;
    const size_t produced = e.run_frames(max_chunk);
    chunk->frames = produced;
    chunk->total_frames = e.seq_frames;
    chunk->ended_by_eos = e.seq_ended ? 1 : 0;
    chunk->status = produced ? QTTS_CHUNK : QTTS_CHUNK_NONE;
    if (produced) {
      const size_t g = e.cfg.cp.groups;
      need(codes_out, "codes_out");
      if (cap < produced * g) qtts::invalid("codes_out capacity too small");
      e.read_codes(before, e.seq_frames, codes_out);
    }
  });
}

void qtts_stream_destroy(qtts_stream* s) { delete s; }

int32_t qtts_text_stream_start(qtts_engine* h, const qtts_generate_options* o,
                               const qtts_text_stream_options* to, qtts_text_stream** out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(o, "options");
    need(out, "out");
    *out = nullptr;
    e.validate(*o);
    qtts_text_stream_options topt;
    qtts_text_stream_options_default(&topt);
    if (to) topt = *to;
    if (topt.min_start_tokens == 0) qtts::invalid("min_start_tokens must be non-zero");
    if (topt.min_resume_tokens == 0) qtts::invalid("min_resume_tokens must be non-zero");
    auto s = std::make_unique<qtts_text_stream>();
    s->s.e = &e;
    s->s.opts = *o;
    s->s.topts = topt;
    *out = s.release();
  });
}

int32_t qtts_text_stream_push_ids(qtts_text_stream* h, const uint32_t* ids, size_t n) {
  return guard([&] {
    need(h, "stream");
    if (h->s.text_finished) qtts::invalid("cannot push text after finish_text");
    if (n) need(ids, "ids");
    h->s.e->check_ids(ids, n);
    for (size_t i = 0; i < n; ++i) h->s.queued.push_back(ids[i]);
  });
}

int32_t qtts_text_stream_finish(qtts_text_stream* h) {
  return guard([&] {
    need(h, "stream");
    if (h->s.text_finished) return;
    h->s.text_finished = true;
    h->s.eos_pending = true;
  });
}

int32_t qtts_text_stream_next_codes_chunk(qtts_text_stream* h, size_t max_chunk,
                                          int32_t* codes_out, size_t cap,
                                          qtts_codes_chunk* chunk) {
  return guard([&] {
    need(h, "stream");
    need(chunk, "chunk");
    qtts::TextStream& s = h->s;
    Engine& e = *s.e;
    QCK(cudaSetDevice(e.device));
    if (max_chunk == 0) qtts::invalid("max_chunk_frames must be non-zero");
    chunk->frames = 0;
    chunk->total_frames = 0;
    chunk->ended_by_eos = 0;
    const size_t G = e.cfg.cp.groups;
    auto finished = [&] {
      s.finished = true;
      chunk->status = QTTS_FINISHED;
      chunk->total_frames = s.codes.size() / G;
      chunk->ended_by_eos = (s.started && e.seq_id == s.id && e.seq_ended) ? 1 : 0;
    };
    if (s.finished) return finished();
    // try_start_generation (generation.rs:1280-1358)
    if (!s.started) {
      bool can = !(s.queued.size() < s.topts.min_start_tokens && !s.text_finished) &&
                 !s.queued.empty();
      if (!can) {
        if (s.text_finished && s.queued.empty() && s.eos_pending) return finished();
        chunk->status = QTTS_NEED_MORE_TEXT;
        return;
      }
      const size_t la = std::max<size_t>(1, std::min<size_t>(s.topts.min_start_tokens, s.queued.size()));
      std::vector<uint32_t> pre;
      for (size_t i = 0; i < la; ++i) {
        pre.push_back(s.queued.front());
        s.queued.pop_front();
      }
      int ntr_unused = 0;
      const int P = e.prepare(pre.data(), pre.size(), pre.size(), s.opts.speaker, s.opts.language,
                              nullptr, &ntr_unused);
      e.begin(P, 0, s.opts);
      s.id = e.seq_id;
      s.started = true;
    }
    if (s.id != e.seq_id) qtts::invalid("text stream was superseded by a newer generation on this engine");
    // next_codes_chunk (generation.rs:1183-1278): plan the trailing rows of the
    // frames this chunk can run, then run them as one burst.
    if (e.seq_ended || (size_t)e.seq_frames >= e.seq_max_frames) {
      return finished();
    }
    std::vector<int> tr_ids;
    size_t n = 0;
    while (n < max_chunk && e.seq_frames + n < e.seq_max_frames) {
      const size_t cur = e.seq_frames + n;
      if (cur + 1 < e.seq_max_frames) {
        const long long id = next_trailing_id(s);
        if (id < 0) break;
        tr_ids.push_back((int)id);
      }
      ++n;
    }
    if (n == 0) {
      chunk->status = QTTS_NEED_MORE_TEXT;
      return;
    }
    const size_t H = e.cfg.talker.hidden;
    if (!tr_ids.empty()) e.project_text(tr_ids, e.trailing + (size_t)e.seq_frames * H);
    const int ntr = e.seq_frames + (int)tr_ids.size();
    e.h2d(&e.st->n_trailing, &ntr, 4);
    QCK(cudaStreamSynchronize(e.stream));
    const size_t before = e.seq_frames;
    const size_t produced = e.run_frames(n);
    if (produced == 0) {
      if (e.seq_ended || (size_t)e.seq_frames >= e.seq_max_frames) return finished();
      chunk->status = QTTS_NEED_MORE_TEXT;
      return;
    }
    const size_t old = s.codes.size();
    s.codes.resize(old + produced * G);
    e.read_codes(before, e.seq_frames, s.codes.data() + old);
    chunk->frames = produced;
    chunk->total_frames = e.seq_frames;
    chunk->ended_by_eos = e.seq_ended ? 1 : 0;
    chunk->status = QTTS_CHUNK;
    if (codes_out) {
      if (cap < produced * G) qtts::invalid("codes_out capacity too small");
      std::memcpy(codes_out, s.codes.data() + old, produced * G * 4);
    }
  });
}

int32_t qtts_text_stream_codes(qtts_text_stream* h, int32_t* codes_out, size_t cap,
                               size_t* frames_out, int32_t* ended) {
  return guard([&] {
    need(h, "stream");
    const size_t G = h->s.e->cfg.cp.groups;
    const size_t frames = h->s.codes.size() / G;
    if (codes_out) {
      if (cap < h->s.codes.size()) qtts::invalid("codes_out capacity too small");
      std::memcpy(codes_out, h->s.codes.data(), h->s.codes.size() * 4);
    }
    if (frames_out) *frames_out = frames;
    if (ended)
      *ended = (h->s.started && h->s.e->seq_id == h->s.id && h->s.e->seq_ended) ? 1 : 0;
  });
}

void qtts_text_stream_destroy(qtts_text_stream* s) { delete s; }

int32_t qtts_talker_prefill(qtts_engine* h, const float* rows, size_t steps, float* hidden_out,
                            float* logits_out, int32_t* token_out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(rows, "rows");
    if (steps == 0) qtts::invalid("prefill steps must be non-zero");
    if (steps > e.max_cache_steps) qtts::invalid("prefill steps outside cache");
    const size_t H = e.cfg.talker.hidden;
    e.h2d(e.tb.x, rows, steps * H * 4);
    qtts_generate_options o;
    qtts_generate_options_default(&o);
    o.do_sample = 0;
    o.max_frames = 1;
    e.begin((int)steps, 0, o);
    if (token_out) *token_out = e.st_host->semantic;
    if (hidden_out) QCK(cudaMemcpy(hidden_out, e.cp_prefix_target(), H * 4, cudaMemcpyDeviceToHost));
    if (logits_out)
      QCK(cudaMemcpy(logits_out, e.logits, e.cfg.talker.vocab * 4, cudaMemcpyDeviceToHost));
  });
}

int32_t qtts_talker_decode_step(qtts_engine* h, const float* input, size_t offset,
                                float* hidden_out, float* logits_out, int32_t* token_out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(input, "input");
    if (offset >= e.max_cache_steps) qtts::invalid("offset outside cache length");
    const size_t H = e.cfg.talker.hidden;
    e.h2d(e.tb.x, input, H * 4);
    e.st_host->talker_pos = (int)offset;
    e.st_host->halt = 0;
    e.st_host->frames = 0;
    e.h2d(e.st, e.st_host, sizeof(qtts::SeqState));
    qtts::SampleCfg greedy{0, 0, 1.f, 1.f};
    e.stack_step(e.talker, e.tb, e.tkv, &e.st->talker_pos, 0, nullptr);
    e.talker_head(qtts::ROLE_TALKER_STEP, e.tb.x, greedy, 1.0f, nullptr, e.cp_prefix_target());
    e.sync_state();
    if (token_out) *token_out = e.st_host->semantic;
    if (hidden_out) QCK(cudaMemcpy(hidden_out, e.cp_prefix_target(), H * 4, cudaMemcpyDeviceToHost));
    if (logits_out)
      QCK(cudaMemcpy(logits_out, e.logits, e.cfg.talker.vocab * 4, cudaMemcpyDeviceToHost));
  });
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Allocation-free talker decode step.
//
// Some hosts embed this library where they may not allocate device memory
// once they are running: a caller that owns a fixed memory budget carved out
// up front (a real-time audio process, a pool-managed serving runtime, or a
// host that forbids cudaMalloc outside start-up because it synchronises the
// device). For them, the talker decode step's per-call working memory -- the
// input row, the QKV projections, the attention output and the MLP
// activations of every layer -- lives in this file-scope device array instead
// of engine-owned memory (the KV cache, weights and logits are the engine's,
// allocated at load). The array is fixed at kStaticScratchBytes and is held by
// every GPU that loads the library until the process exits. All calls share it
// and it keeps the last call's contents; calls that overlap on the GPU (two
// streams, two engines, two threads) race on it and must be serialised by the
// caller.
// ---------------------------------------------------------------------------
namespace {

constexpr size_t kStaticScratchBytes = 270336;  // 264 KiB
static __device__ __align__(256) float g_step_scratch[kStaticScratchBytes / sizeof(float)];

std::mutex g_static_mu;
void* g_static_ptr[128] = {};

// First call per device (with that device current) resolves the array's
// device address; host code may not use the symbol itself as a pointer.
void* static_scratch_for_device(int device) {
  std::lock_guard<std::mutex> lock(g_static_mu);
  if (device < 0 || device >= 128) qtts::invalid("device index out of range");
  if (!g_static_ptr[device]) {
    void* ptr = nullptr;
    QCK(cudaGetSymbolAddress(&ptr, g_step_scratch));
    g_static_ptr[device] = ptr;
  }
  return g_static_ptr[device];
}

}  // namespace

extern "C" {

int32_t qtts_talker_decode_step_static(qtts_engine* h, const float* input, size_t offset,
                                       float* hidden_out, float* logits_out,
                                       int32_t* token_out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(input, "input");
    if (offset >= e.max_cache_steps) qtts::invalid("offset outside cache length");
    const auto& c = e.talker.c;
    qtts::DevStack& S = e.talker;
    const size_t H = c.hidden;
    // step activations, each 64-float aligned: x, qkv, attention, h1, MLP
    auto up = [](size_t n) { return (n + 63) / 64 * 64; };
    const size_t nx = up(H), nqkv = up(S.qkv_w), nattn = up(S.q_out), nh1 = up(H),
                 nact = up(c.intermediate), nq = e.kv_form() ? up(S.q_out) : 0;
    const size_t need_bytes = (nx + nqkv + nattn + nh1 + nact + nq) * sizeof(float);
    if (need_bytes > kStaticScratchBytes)
      qtts::invalid("talker step needs " + std::to_string(need_bytes) +
                    " bytes of activations; the static array holds " +
                    std::to_string(kStaticScratchBytes));
    float* base = static_cast<float*>(static_scratch_for_device(e.device));
    qtts::StackBufs B{};
    B.x = base;
    B.qkv = B.x + nx;
    B.attn = B.qkv + nqkv;
    B.h1 = B.attn + nattn;
    B.act = B.h1 + nh1;
    B.q = B.act + nact;
    e.h2d(B.x, input, H * 4);
    e.st_host->talker_pos = (int)offset;
    e.st_host->halt = 0;
    e.st_host->frames = 0;
    e.h2d(e.st, e.st_host, sizeof(qtts::SeqState));
    // The same layer sequence as qtts_talker_decode_step, over the static
    // array (the engine's other workspaces were allocated at load).
    e.stack_step(S, B, e.tkv, &e.st->talker_pos, 0, nullptr);
    qtts::SampleCfg greedy{0, 0, 1.f, 1.f};
    e.talker_head(qtts::ROLE_TALKER_STEP, B.x, greedy, 1.0f, nullptr, e.cp_prefix_target());
    e.sync_state();
    if (token_out) *token_out = e.st_host->semantic;
    if (hidden_out) QCK(cudaMemcpy(hidden_out, e.cp_prefix_target(), H * 4, cudaMemcpyDeviceToHost));
    if (logits_out)
      QCK(cudaMemcpy(logits_out, e.logits, c.vocab * 4, cudaMemcpyDeviceToHost));
  });
}

int32_t qtts_code_predictor(qtts_engine* h, const float* talker_hidden, const float* semantic_embed,
                            const qtts_generate_options* o, int32_t* tokens_out,
                            float* emb_sum_out, float* logits_out) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(talker_hidden, "talker_hidden");
    need(semantic_embed, "semantic_embed");
    need(o, "options");
    qtts_generate_options opt = *o;
    opt.decode_audio = 0;
    opt.max_frames = 1;
    e.validate(opt);
    const size_t H = e.cfg.talker.hidden;
    const auto& C = e.cfg.cp;
    e.h2d(e.cp_prefix_target(), talker_hidden, H * 4);
    e.h2d(e.cp_prefix_target() + H, semantic_embed, H * 4);
    qtts::SeqState s{};
    s.semantic = 0;
    s.rng_kind = opt.rng;
    s.rng_state = opt.seed ^ qtts::kSeedXor;
    s.rng_seed = opt.seed;
    s.n_trailing = 0;
    *e.st_host = s;
    e.h2d(e.st, e.st_host, sizeof(s));
    const qtts::SampleCfg sc = qtts::sub_cfg(opt);
    const int na = C.groups - 1;
    // Eager CodePredictor pass with per-group logits kept for parity checks.
    if (e.has_proj())
      e.linear(e.proj_w, e.cp_prefix, H, nullptr, 0.f, e.cb.x, C.hidden, nullptr, 0, e.proj_b, 2,
               C.hidden, H, qtts::EPI_BIAS, nullptr);
    e.stack_rows(e.cp, e.cb, e.ckv, 2, 0, nullptr);
    e.cp_head(0, e.cb.x + C.hidden, sc, nullptr);
    QCK(cudaMemcpyAsync(e.dbg_logits, e.logits, C.vocab * 4, cudaMemcpyDeviceToDevice, e.stream));
    for (int g = 1; g < C.groups - 1; ++g) {
      if (e.has_proj() && !e.cp_x0)
        e.linear(e.proj_w, e.cp_next, H, nullptr, 0.f, e.cb.x, C.hidden, nullptr, 0, e.proj_b, 1,
                 C.hidden, H, qtts::EPI_BIAS, nullptr);
      e.stack_step(e.cp, e.cb, e.ckv, nullptr, g + 1, nullptr, e.cp_qkv0 != nullptr);
      e.cp_head(g, e.cb.x, sc, nullptr);
      QCK(cudaMemcpyAsync(e.dbg_logits + (size_t)g * C.vocab, e.logits, C.vocab * 4,
                                cudaMemcpyDeviceToDevice, e.stream));
    }
    e.sync_state();
    std::vector<int32_t> row(C.groups);
    e.read_codes(0, 1, row.data());
    if (tokens_out) std::memcpy(tokens_out, row.data() + 1, na * 4);
    if (emb_sum_out) QCK(cudaMemcpy(emb_sum_out, e.emb_sum, H * 4, cudaMemcpyDeviceToHost));
    if (logits_out)
      QCK(cudaMemcpy(logits_out, e.dbg_logits, (size_t)na * C.vocab * 4, cudaMemcpyDeviceToHost));
    e.seq_ended = true;  // the talker state was not advanced: no stream may continue
    ++e.seq_id;
  });
}

int32_t qtts_step_trace_enable(qtts_engine* h, int32_t on) {
  return guard([&] {
    Engine& e = engine_of(h);
    if (e.trace_on == (on != 0)) return;
    e.trace_on = on != 0;
    // the frame graphs carry the trace ids fixed at capture: recapture
    QCK(cudaStreamSynchronize(e.stream));
    for (auto& kv : e.graphs) cudaGraphExecDestroy(kv.second);
    e.graphs.clear();
    e.trace_rows.clear();
  });
}

int32_t qtts_step_trace_read(const qtts_engine* h, qtts_trace_launch* out, size_t cap,
                             size_t* n) {
  return guard([&] {
    need(h, "engine");
    need(n, "n");
    const Engine& e = *h->e;
    *n = e.trace_rows.size();
    if (out) std::memcpy(out, e.trace_rows.data(), std::min(cap, *n) * sizeof(qtts_trace_launch));
  });
}

int32_t qtts_selftest_device_wait(qtts_engine* h, uint32_t limit_us) {
  return guard([&] {
    Engine& e = engine_of(h);
    if (limit_us == 0 || limit_us > 5000000u) qtts::invalid("limit_us must be in (0, 5e6]");
    // a private counter nobody increments, and the wait's status word
    if (!e.selftest_ctr) {
      e.selftest_ctr = e.arena.alloc<unsigned long long>(1);
      e.selftest_status = e.arena.alloc<int>(1);
    }
    unsigned long long* ctr = e.selftest_ctr;
    int* status = e.selftest_status;
    QCK(cudaMemsetAsync(ctr, 0, sizeof(unsigned long long), e.stream));
    QCK(cudaMemsetAsync(status, 0xff, sizeof(int), e.stream));
    QCK(qtts::launch_wait_selftest(ctr, 1ull, (unsigned long long)limit_us * 1000ull, status,
                                   e.stream));
    int st = -1;
    QCK(cudaMemcpyAsync(&st, status, sizeof(int), cudaMemcpyDeviceToHost, e.stream));
    e.stream_sync();
    if (st == 1)
      qtts::fail(QTTS_ERR_DEVICE_STATE, "a bounded device wait ran out after " +
                                            std::to_string(limit_us) + " us");
    if (st != 0) qtts::fail(QTTS_ERR_CUDA, "wait self-test did not report");
  });
}

int32_t qtts_last_launch_count(const qtts_engine* h, size_t* kernels) {
  return guard([&] {
    need(h, "engine");
    need(kernels, "kernels");
    *kernels = h->e->last_launches;
  });
}

int32_t qtts_profile_projection(qtts_engine* h, int32_t which, int32_t n_launch,
                                float* ms_per_launch, double* bytes_per_launch) {
  return guard([&] {
    Engine& e = engine_of(h);
    need(ms_per_launch, "ms_per_launch");
    if (n_launch <= 0) qtts::invalid("launches must be positive");
    qtts::DevStack& S = e.talker;
    const auto& c = S.c;
    const qtts::StackBufs& B = e.tb;
    double bytes = 0;
    auto one = [&](int l) {
      switch (which) {
        case 0:  // gate|up + SwiGLU, RMSNorm prologue
          e.linear(S.wgu[l], B.h1, c.hidden, S.post_g[l], c.eps, B.act, c.intermediate, nullptr, 0,
                   nullptr, 1, c.intermediate, c.hidden, qtts::EPI_SWIGLU, nullptr);
          bytes = 2.0 * c.intermediate * c.hidden * 2 + 4.0 * (c.hidden * 2 + c.intermediate);
          break;
        case 1:  // QKV, RMSNorm prologue
          e.linear(S.wqkv[l], B.x, c.hidden, S.in_g[l], c.eps, B.qkv, S.qkv_w, nullptr, 0, nullptr,
                   1, S.qkv_w, c.hidden, qtts::EPI_STORE, nullptr);
          bytes = 2.0 * S.qkv_w * c.hidden + 4.0 * (c.hidden * 2 + S.qkv_w);
          break;
        case 2:  // down + residual
          e.linear(S.wdown[l], B.act, c.intermediate, nullptr, 0.f, B.q, c.hidden, B.h1, c.hidden,
                   nullptr, 1, c.hidden, c.intermediate, qtts::EPI_RESID, nullptr);
          bytes = 2.0 * c.hidden * c.intermediate + 4.0 * (c.intermediate + 2 * c.hidden);
          break;
        default:  // O + residual
          e.linear(S.wo[l], B.attn, S.q_out, nullptr, 0.f, B.q, c.hidden, B.x, c.hidden, nullptr, 1,
                   c.hidden, S.q_out, qtts::EPI_RESID, nullptr);
          bytes = 2.0 * c.hidden * S.q_out + 4.0 * (S.q_out + 2 * c.hidden);
      }
    };
    // Cycle through every layer's weights so each launch streams from HBM
    // (28 distinct matrices exceed the 126 MB L2).
    for (int i = 0; i < c.layers; ++i) one(i);
    QCK(cudaEventRecord(e.ev1, e.stream));
    for (int i = 0; i < n_launch; ++i) one(i % c.layers);
    QCK(cudaEventRecord(e.ev2, e.stream));
    QCK(cudaEventSynchronize(e.ev2));
    float ms = 0.f;
    QCK(cudaEventElapsedTime(&ms, e.ev1, e.ev2));
    *ms_per_launch = ms / n_launch;
    if (bytes_per_launch) *bytes_per_launch = bytes;
  });
}

int32_t qtts_last_timings(const qtts_engine* h, float* prefill_ms, float* frames_ms,
                          size_t* frames) {
  return guard([&] {
    need(h, "engine");
    if (prefill_ms) *prefill_ms = h->e->last_prefill_ms;
    if (frames_ms) *frames_ms = h->e->last_frames_ms;
    if (frames) *frames = h->e->last_frames;
  });
}

}  // extern "C"
