// PyTorch-ROCm extension: the reference's pybind classes over the C ABI of libqwentts_amd.
//
// MegakernelTTSDecoder           -- qwentts_turbo/megakernel_backbone.py:109-332
// MegakernelCodePredictorDecoder -- qwentts_turbo/megakernel_code_predictor.py:86-242
//
// Same constructor arguments, method names and return conventions as the reference (outputs
// are fresh tensors; KV getters alias the internal caches). Differences: shapes, dtypes,
// devices and positions are validated (the reference checks nothing), launch errors raise,
// and extra methods expose the fused head / token-selection / frame entry points.
#include <torch/extension.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <hip/hip_runtime_api.h>
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>
#include <vector>
#include "qwentts_amd.h"

namespace {

constexpr int kHidden = 1024, kKVHeads = 8, kHeadDim = 128, kInter = 3072, kQ = 2048;
constexpr int kMaxStreams = 8;   // streams of one frames_streams() launch (one per XCD)

hipStream_t cur_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

void hip_check(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, " failed: ", hipGetErrorString(e));
}

void check_bf16(const torch::Tensor& t, std::vector<int64_t> shape, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bfloat16, got ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.sizes().vec() == shape, name, " has shape ", t.sizes(), ", expected ", c10::IntArrayRef(shape));
}

// Layer weights in the reference's struct order (11 per layer).
std::vector<TTSLayerWeights> pack_layers(const std::vector<torch::Tensor>& flat, int num_layers) {
  TORCH_CHECK((int)flat.size() == num_layers * 11, "expected ", num_layers * 11, " layer weights, got ", flat.size());
  const std::vector<std::vector<int64_t>> shapes = {
      {kHidden}, {kQ, kHidden}, {kKVHeads * kHeadDim, kHidden}, {kKVHeads * kHeadDim, kHidden},
      {kHeadDim}, {kHeadDim}, {kHidden, kQ}, {kHidden}, {kInter, kHidden}, {kInter, kHidden}, {kHidden, kInter}};
  std::vector<TTSLayerWeights> out(num_layers);
  for (int i = 0; i < num_layers; ++i) {
    const void** p = reinterpret_cast<const void**>(&out[i]);
    for (int j = 0; j < 11; ++j) {
      const auto& t = flat[i * 11 + j];
      check_bf16(t, shapes[j], "layer weight");
      TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0, "layer weights must be 16-byte aligned");
      p[j] = t.data_ptr();
    }
  }
  return out;
}

torch::Tensor upload_struct(const void* data, size_t bytes, const torch::Device& dev) {
  auto t = torch::empty({(int64_t)bytes}, torch::dtype(torch::kUInt8).device(dev));
  hip_check(hipMemcpy(t.data_ptr(), data, bytes, hipMemcpyHostToDevice), "hipMemcpy");
  return t;
}

torch::Tensor make_workspace(const torch::Device& dev) {
  auto ws = torch::zeros({(int64_t)qtts_workspace_bytes()}, torch::dtype(torch::kUInt8).device(dev));
  hip_check(qtts_workspace_init(ws.data_ptr(), dev.index()), "qtts_workspace_init (needs an MI355X: gfx950, 256 CUs)");
  return ws;
}

torch::Tensor as_bf16_vec(torch::Tensor e, const torch::Device& dev) {
  if (e.dim() == 2) e = e.squeeze(0);
  TORCH_CHECK(e.dim() == 1 && e.size(0) == kHidden, "input embedding must be [1024] or [1, 1024], got ", e.sizes());
  TORCH_CHECK(e.device() == dev, "input embedding must be on ", dev);
  return e.to(torch::kBFloat16).contiguous();
}

QttsSampling sampling(bool do_sample, double temperature, int64_t top_k, double top_p, int64_t seed) {
  TORCH_CHECK(!do_sample || temperature > 0.0, "temperature must be > 0");
  QttsSampling s;
  s.do_sample = do_sample ? 1 : 0;
  s.temperature = (float)temperature;
  s.top_k = (int)top_k;
  s.top_p = (float)top_p;
  s.seed = (unsigned long long)seed;
  return s;
}

// the weight-shared launches' workspace, allocated on first use (its first launch zero-fills it)
void ensure_shared_ws(torch::Tensor& ws, const torch::Device& dev) {
  if (ws.defined()) return;
  ws = torch::empty({(int64_t)qtts_shared_workspace_bytes()}, torch::dtype(torch::kUInt8).device(dev));
  hip_check(qtts_workspace_init(ws.data_ptr(), dev.index()), "qtts_workspace_init");
}
void check_shared_error(const torch::Tensor& ws) {
  if (!ws.defined()) return;
  unsigned int code = 0;
  hip_check(qtts_shared_workspace_check(ws.data_ptr(), &code, cur_stream()), "qtts_shared_workspace_check");
  TORCH_CHECK(code == 0, "weight-shared decode kernel reported a device-side wait timeout (error word ", code, ")");
}

void check_device_error(const torch::Tensor& ws) {
  unsigned int code = 0;
  hip_check(qtts_workspace_check(ws.data_ptr(), &code, cur_stream()), "qtts_workspace_check");
  TORCH_CHECK(code == 0, "decode kernel reported a device-side wait timeout (error word ", code, ")");
}

// ---------------------------------------------------------------------------------------
class MegakernelTTSDecoder {
 public:
  MegakernelTTSDecoder(torch::Tensor embed_weight, std::vector<torch::Tensor> layer_weights_flat,
                       torch::Tensor final_norm_weight, torch::Tensor codec_head_weight, torch::Tensor cos_table,
                       torch::Tensor sin_table, int64_t num_layers, int64_t max_seq_len)
      : num_layers_((int)num_layers), max_seq_len_((int)max_seq_len), dev_(embed_weight.device()) {
    TORCH_CHECK(num_layers >= 1, "num_layers must be >= 1");
    TORCH_CHECK(max_seq_len >= 1, "max_seq_len must be >= 1");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    TORCH_CHECK(embed_weight.dim() == 2 && embed_weight.size(1) == kHidden, "embed_weight must be [vocab, 1024]");
    check_bf16(embed_weight, {embed_weight.size(0), kHidden}, "embed_weight");
    check_bf16(codec_head_weight, {codec_head_weight.size(0), kHidden}, "codec_head_weight");
    check_bf16(final_norm_weight, {kHidden}, "final_norm_weight");
    TORCH_CHECK(cos_table.size(0) >= max_seq_len && sin_table.size(0) >= max_seq_len, "RoPE tables shorter than max_seq_len");
    check_bf16(cos_table, {cos_table.size(0), kHeadDim}, "cos_table");
    check_bf16(sin_table, {sin_table.size(0), kHeadDim}, "sin_table");
    embed_weight_ = embed_weight;
    final_norm_weight_ = final_norm_weight;
    codec_head_weight_ = codec_head_weight;
    cos_table_ = cos_table;
    sin_table_ = sin_table;
    layer_weights_tensors_ = layer_weights_flat;
    auto host = pack_layers(layer_weights_flat, num_layers_);
    d_layer_weights_ = upload_struct(host.data(), host.size() * sizeof(TTSLayerWeights), dev_);
    auto bf = torch::dtype(torch::kBFloat16).device(dev_);
    auto f32 = torch::dtype(torch::kFloat32).device(dev_);
    k_cache_ = torch::zeros({num_layers, kKVHeads, max_seq_len, kHeadDim}, bf);
    v_cache_ = torch::zeros({num_layers, kKVHeads, max_seq_len, kHeadDim}, bf);
    hidden_buffer_ = torch::zeros({kHidden}, bf);
    g_normalized_ = torch::zeros({kHidden}, f32);
    logits_ = torch::zeros({codec_head_weight.size(0)}, f32);
    token_ = torch::zeros({1}, torch::dtype(torch::kInt32).device(dev_));
    ws_ = make_workspace(dev_);
    position_ = 0;
  }
  ~MegakernelTTSDecoder() {
    (void)qtts_workspace_release(ws_.data_ptr(), 1);
    if (ws_streams_.defined()) (void)qtts_workspace_release(ws_streams_.data_ptr(), kMaxStreams);
    if (ws_shared_.defined()) (void)qtts_workspace_release(ws_shared_.data_ptr(), 1);
  }
  MegakernelTTSDecoder(const MegakernelTTSDecoder&) = delete;
  MegakernelTTSDecoder& operator=(const MegakernelTTSDecoder&) = delete;

  torch::Tensor decode_step(int64_t input_token_id) {
    TORCH_CHECK(input_token_id >= 0 && input_token_id < embed_weight_.size(0), "token id out of range");
    run(nullptr, (int)input_token_id, nullptr, false, nullptr, 0, 1.0, -1, false, sampling(false, 1.0, 0, 1.0, 0), 0);
    return g_normalized_.clone();
  }

  int64_t decode_step_with_argmax(int64_t input_token_id) {
    TORCH_CHECK(input_token_id >= 0 && input_token_id < embed_weight_.size(0), "token id out of range");
    run(nullptr, (int)input_token_id, nullptr, true, nullptr, 0, 1.0, -1, false, sampling(false, 1.0, 0, 1.0, 0), 0,
        /*no_mask=*/true);
    return token_.item<int>();
  }

  torch::Tensor decode_step_with_embedding(torch::Tensor input_embedding) {
    auto e = as_bf16_vec(input_embedding, dev_);
    run(e.data_ptr(), 0, nullptr, false, nullptr, 0, 1.0, -1, false, sampling(false, 1.0, 0, 1.0, 0), 0);
    return g_normalized_.clone();
  }

  // Extended: one step with 3D rotary positions (t, h, w); returns the final hidden.
  torch::Tensor decode_step_3d(torch::Tensor input_embedding, std::vector<int64_t> pos3) {
    TORCH_CHECK(pos3.size() == 3, "pos3 must be (t, h, w)");
    auto e = as_bf16_vec(input_embedding, dev_);
    int p3[3] = {(int)pos3[0], (int)pos3[1], (int)pos3[2]};
    run(e.data_ptr(), 0, p3, false, nullptr, 0, 1.0, -1, false, sampling(false, 1.0, 0, 1.0, 0), 0);
    return g_normalized_.clone();
  }

  // Extended: step + fused codec head + on-device selection. Writes the token to
  // out_token (int32 [1] device); keeps hidden / logits in the internal buffers.
  void decode_step_select(torch::Tensor input_embedding, torch::Tensor out_token, torch::Tensor history,
                          int64_t n_history, double repetition_penalty, int64_t eos_id, bool suppress_eos,
                          bool do_sample, double temperature, int64_t top_k, double top_p, int64_t seed,
                          int64_t frame_step, c10::optional<std::vector<int64_t>> pos3, c10::optional<torch::Tensor> skip_if) {
    auto e = as_bf16_vec(input_embedding, dev_);
    TORCH_CHECK(out_token.is_cuda() && out_token.scalar_type() == torch::kInt32 && out_token.numel() >= 1,
                "out_token must be an int32 GPU tensor");
    TORCH_CHECK(history.is_cuda() && history.scalar_type() == torch::kInt32 && history.numel() >= n_history,
                "history must be an int32 GPU tensor with >= n_history entries");
    int p3[3];
    int* p3p = nullptr;
    if (pos3.has_value()) {
      TORCH_CHECK(pos3->size() == 3, "pos3 must be (t, h, w)");
      for (int i = 0; i < 3; ++i) p3[i] = (int)(*pos3)[i];
      p3p = p3;
    }
    const int* skip = nullptr;
    if (skip_if.has_value()) {
      TORCH_CHECK(skip_if->is_cuda() && skip_if->scalar_type() == torch::kInt32, "skip_if must be an int32 GPU tensor");
      skip = skip_if->data_ptr<int>();
    }
    run(e.data_ptr(), 0, p3p, true, history.data_ptr<int>(), (int)n_history, repetition_penalty, (int)eos_id, suppress_eos,
        sampling(do_sample, temperature, top_k, top_p, seed), (int)frame_step, false, out_token.data_ptr<int>(), skip);
  }

  // Extended: prefill of the prompt embeddings [S, 1024] at positions position() .. position() + S - 1
  // in one call (qtts_backbone_prefill: the transformers bf16 forward on MFMA, K/V straight into
  // this decoder's cache). Returns the last token's final-norm hidden (f32 [1024] of bf16 values),
  // also left in hidden_state_buffer(). With out_token, the first group-0 token is selected from
  // the codec head (suppress mask, EOS removed when suppress_eos; generator.py:113-119). pos3:
  // optional int32 [3, S] rotary (t, h, w) rows. The position advances by S.
  torch::Tensor prefill(torch::Tensor embeds, c10::optional<torch::Tensor> out_token, int64_t eos_id, bool suppress_eos,
                        bool do_sample, double temperature, int64_t top_k, double top_p, int64_t seed,
                        c10::optional<torch::Tensor> pos3) {
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    if (embeds.dim() == 3) embeds = embeds.squeeze(0);
    TORCH_CHECK(embeds.dim() == 2 && embeds.size(1) == kHidden && embeds.size(0) >= 1, "embeds must be [S, 1024], got ",
                embeds.sizes());
    TORCH_CHECK(embeds.device() == dev_, "embeds must be on ", dev_);
    auto e = embeds.to(torch::kBFloat16).contiguous();
    const int S = (int)e.size(0);
    TORCH_CHECK(position_ + S <= max_seq_len_, "prefill of ", S, " tokens at position ", position_, " exceeds max_seq_len ",
                max_seq_len_);
    const int* p3 = nullptr;
    torch::Tensor p3t;
    if (pos3.has_value()) {
      p3t = pos3->to(dev_, torch::kInt32).contiguous();
      TORCH_CHECK(p3t.dim() == 2 && p3t.size(0) == 3 && p3t.size(1) == S, "pos3 must be [3, S]");
      p3 = p3t.data_ptr<int>();
    }
    int* tok = nullptr;
    if (out_token.has_value()) {
      TORCH_CHECK(out_token->is_cuda() && out_token->scalar_type() == torch::kInt32 && out_token->numel() >= 1,
                  "out_token must be an int32 GPU tensor");
      tok = out_token->data_ptr<int>();
    }
    const int vocab = (int)codec_head_weight_.size(0);
    const size_t need = qtts_prefill_workspace_bytes(S, tok ? vocab : 0);
    TORCH_CHECK(need > 0, "prefill workspace size query failed");
    if (!pf_ws_.defined() || (size_t)pf_ws_.numel() < need)
      pf_ws_ = torch::empty({(int64_t)need}, torch::dtype(torch::kUInt8).device(dev_));
    QttsSampling samp = sampling(do_sample, temperature, top_k, top_p, seed);
    hip_check(qtts_backbone_prefill(pf_ws_.data_ptr(), (size_t)pf_ws_.numel(),
                                    reinterpret_cast<const TTSLayerWeights*>(d_layer_weights_.data_ptr()), num_layers_,
                                    final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(),
                                    k_cache_.data_ptr(), v_cache_.data_ptr(), max_seq_len_, position_, S, p3, e.data_ptr(),
                                    g_normalized_.data_ptr<float>(), tok ? codec_head_weight_.data_ptr() : nullptr, vocab,
                                    tok ? logits_.data_ptr<float>() : nullptr, tok, 1, (int)eos_id, suppress_eos ? 1 : 0,
                                    &samp, 0, cur_stream()),
              "qtts_backbone_prefill");
    position_ += S;
    return g_normalized_.clone();
  }

  // Extended: decode_step_select for up to 8 independent decoders `decs` (sharing this decoder's
  // weights) in one launch, decoder s on XCD s, each at its own position with its own KV cache.
  // out_tokens[s] gets stream s's token and hidden_out[s] (f32 [n, 1024]) its final-norm hidden;
  // the residual and logits go to each decoder's own buffers. Stream s samples with key seed + s
  // and applies the repetition penalty over history[s][0 : n_history[s]]. Each position advances
  // by one. The launch uses this decoder's block of per-stream workspaces.
  void decode_steps_streams(std::vector<MegakernelTTSDecoder*> decs, torch::Tensor embeds, torch::Tensor out_tokens,
                            torch::Tensor hidden_out, c10::optional<torch::Tensor> history, std::vector<int64_t> n_history,
                            double repetition_penalty, int64_t eos_id, bool suppress_eos, bool do_sample,
                            double temperature, int64_t top_k, double top_p, int64_t seed, int64_t frame_step,
                            c10::optional<torch::Tensor> skip, bool shared) {
    const int64_t n = (int64_t)decs.size();
    TORCH_CHECK(n >= 1 && n <= kMaxStreams, "decode_steps_streams takes 1..", kMaxStreams, " decoders, got ", n);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    check_bf16(embeds, {n, kHidden}, "embeds");
    TORCH_CHECK(embeds.device() == dev_, "embeds must be on ", dev_);
    TORCH_CHECK(out_tokens.is_cuda() && out_tokens.scalar_type() == torch::kInt32 && out_tokens.is_contiguous() &&
                    out_tokens.numel() >= n, "out_tokens must be a contiguous int32 GPU tensor with >= ", n, " entries");
    TORCH_CHECK(hidden_out.is_cuda() && hidden_out.scalar_type() == torch::kFloat32 && hidden_out.is_contiguous() &&
                    hidden_out.sizes() == torch::IntArrayRef({n, kHidden}), "hidden_out must be a contiguous f32 [", n, ", 1024] GPU tensor");
    TORCH_CHECK(n_history.empty() || (int64_t)n_history.size() == n, "n_history needs one entry per decoder");
    int64_t hist_stride = 0;
    if (history.has_value()) {
      TORCH_CHECK(history->is_cuda() && history->scalar_type() == torch::kInt32 && history->is_contiguous() &&
                      history->dim() == 2 && history->size(0) >= n, "history must be a contiguous int32 [n, H] GPU tensor");
      hist_stride = history->size(1);
    }
    if (skip.has_value())
      TORCH_CHECK(skip->is_cuda() && skip->scalar_type() == torch::kInt32 && skip->is_contiguous() && skip->numel() >= n,
                  "skip must be a contiguous int32 GPU tensor with >= ", n, " entries");
    std::vector<QttsBackboneStream> io(n);
    for (int64_t st = 0; st < n; ++st) {
      MegakernelTTSDecoder* d = decs[st];
      TORCH_CHECK(d != nullptr, "decoder ", st, " is None");
      TORCH_CHECK(d->dev_ == dev_ && d->num_layers_ == num_layers_ && d->max_seq_len_ == max_seq_len_ &&
                      d->layer_weights_tensors_.size() == layer_weights_tensors_.size() &&
                      d->codec_head_weight_.data_ptr() == codec_head_weight_.data_ptr() &&
                      d->final_norm_weight_.data_ptr() == final_norm_weight_.data_ptr() &&
                      d->cos_table_.data_ptr() == cos_table_.data_ptr() && d->sin_table_.data_ptr() == sin_table_.data_ptr(),
                  "decoder ", st, " does not share this decoder's weights");
      for (size_t j = 0; j < layer_weights_tensors_.size(); ++j)
        TORCH_CHECK(d->layer_weights_tensors_[j].data_ptr() == layer_weights_tensors_[j].data_ptr(),
                    "decoder ", st, " does not share this decoder's layer weights");
      for (int64_t o = 0; o < st; ++o) TORCH_CHECK(decs[o] != d, "decoder ", st, " appears twice");
      TORCH_CHECK(d->position_ < max_seq_len_, "decoder ", st, ": position ", d->position_, " >= max_seq_len ",
                  max_seq_len_, " (KV cache full)");
      const int nh = n_history.empty() ? 0 : (int)n_history[st];
      TORCH_CHECK(nh >= 0 && nh <= hist_stride, "n_history[", st, "] = ", nh, " outside [0, ", hist_stride, "]");
      QttsBackboneStream& q = io[st];
      q.k_cache = d->k_cache_.data_ptr();
      q.v_cache = d->v_cache_.data_ptr();
      q.position = d->position_;
      q.pos3[0] = q.pos3[1] = q.pos3[2] = d->position_;
      q.input_embedding = static_cast<const uint16_t*>(embeds.data_ptr()) + st * kHidden;
      q.out_hidden = hidden_out.data_ptr<float>() + st * kHidden;
      q.out_residual = d->hidden_buffer_.data_ptr();
      q.out_logits = d->logits_.data_ptr<float>();
      q.out_token = out_tokens.data_ptr<int>() + st;
      q.history = nh > 0 ? history->data_ptr<int>() + st * hist_stride : nullptr;
      q.n_history = nh;
      q.seed = (unsigned long long)(seed + st);
      q.skip_if = skip.has_value() ? skip->data_ptr<int>() + st : nullptr;
    }
    QttsSampling samp = sampling(do_sample, temperature, top_k, top_p, seed);
    if (shared) {
      ensure_shared_ws(ws_shared_, dev_);
      hip_check(qtts_backbone_step_shared((int)n, ws_shared_.data_ptr(), reinterpret_cast<const TTSLayerWeights*>(d_layer_weights_.data_ptr()),
                                          num_layers_, final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(),
                                          max_seq_len_, io.data(), codec_head_weight_.data_ptr(), (int)codec_head_weight_.size(0),
                                          1, (float)repetition_penalty, (int)eos_id, suppress_eos ? 1 : 0, &samp, (int)frame_step,
                                          cur_stream()),
                "qtts_backbone_step_shared");
      for (auto* d : decs) d->position_++;
      return;
    }
    if (!ws_streams_.defined()) {
      ws_streams_ = torch::zeros({(int64_t)(kMaxStreams * qtts_workspace_bytes())}, torch::dtype(torch::kUInt8).device(dev_));
      hip_check(qtts_workspace_init(ws_streams_.data_ptr(), dev_.index()), "qtts_workspace_init");
    }
    hip_check(qtts_backbone_step_streams((int)n, ws_streams_.data_ptr(), reinterpret_cast<const TTSLayerWeights*>(d_layer_weights_.data_ptr()),
                                         num_layers_, final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(),
                                         max_seq_len_, io.data(), codec_head_weight_.data_ptr(), (int)codec_head_weight_.size(0),
                                         1, (float)repetition_penalty, (int)eos_id, suppress_eos ? 1 : 0, &samp, (int)frame_step,
                                         cur_stream()),
              "qtts_backbone_step_streams");
    for (auto* d : decs) d->position_++;
  }
  // the wait-timeout error words of the decode_steps_streams() workspaces
  void check_error_streams() const {
    check_shared_error(ws_shared_);
    if (!ws_streams_.defined()) return;
    for (int st = 0; st < kMaxStreams; ++st) {
      unsigned int code = 0;
      hip_check(qtts_workspace_check(static_cast<uint8_t*>(ws_streams_.data_ptr()) + st * qtts_workspace_bytes(), &code, cur_stream()),
                "qtts_workspace_check");
      TORCH_CHECK(code == 0, "decode kernel reported a device-side wait timeout in stream ", st, " (error word ", code, ")");
    }
  }

  void reset() {
    position_ = 0;
    k_cache_.zero_();
    v_cache_.zero_();
  }
  int64_t position() const { return position_; }
  void set_position(int64_t pos) {
    TORCH_CHECK(pos >= 0 && pos <= max_seq_len_, "position ", pos, " outside [0, ", max_seq_len_, "]");
    position_ = (int)pos;
  }
  torch::Tensor get_hidden_states() const { return g_normalized_.clone(); }
  torch::Tensor get_k_cache() const { return k_cache_; }
  torch::Tensor get_v_cache() const { return v_cache_; }
  torch::Tensor hidden_state_buffer() const { return g_normalized_; }
  torch::Tensor residual_buffer() const { return hidden_buffer_; }
  torch::Tensor logits_buffer() const { return logits_; }
  void check_error() const { check_device_error(ws_); }
  // test hook: pre-sets the workspace's error word (after at least one launch), so that every
  // wait of the next launch gives up at its first check
  void debug_set_error(int64_t code) {
    hip_check(qtts_debug_set_error(ws_.data_ptr(), (unsigned int)code, cur_stream()), "qtts_debug_set_error");
  }

  void set_kv_cache(torch::Tensor k_cache, torch::Tensor v_cache) {
    TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(), "k/v must be [layers, 8, seq, 128]");
    TORCH_CHECK(k_cache.size(0) == num_layers_ && k_cache.size(1) == kKVHeads && k_cache.size(3) == kHeadDim,
                "k/v must be [", num_layers_, ", 8, seq, 128], got ", k_cache.sizes());
    TORCH_CHECK(k_cache.size(2) <= max_seq_len_, "k/v longer than max_seq_len");
    using namespace torch::indexing;
    k_cache_.index_put_({Slice(), Slice(), Slice(0, k_cache.size(2)), Slice()}, k_cache.to(dev_, torch::kBFloat16));
    v_cache_.index_put_({Slice(), Slice(), Slice(0, v_cache.size(2)), Slice()}, v_cache.to(dev_, torch::kBFloat16));
  }

 private:
  void run(const void* emb, int token, const int* pos3, bool with_head, const int* history, int n_history,
           double rep_penalty, int eos_id, bool suppress_eos, QttsSampling samp, int frame_step, bool no_mask = false,
           int* out_token = nullptr, const int* skip = nullptr) {
    TORCH_CHECK(position_ < max_seq_len_, "position ", position_, " >= max_seq_len ", max_seq_len_, " (KV cache full)");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    const int vocab = (int)codec_head_weight_.size(0);
    int* tok = out_token ? out_token : token_.data_ptr<int>();
    hipError_t e = qtts_backbone_step(
        ws_.data_ptr(), reinterpret_cast<const TTSLayerWeights*>(d_layer_weights_.data_ptr()), num_layers_,
        final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(), k_cache_.data_ptr(),
        v_cache_.data_ptr(), max_seq_len_, position_, pos3, emb, emb ? nullptr : embed_weight_.data_ptr(), token,
        g_normalized_.data_ptr<float>(), hidden_buffer_.data_ptr(), with_head ? codec_head_weight_.data_ptr() : nullptr,
        vocab, with_head ? logits_.data_ptr<float>() : nullptr, with_head ? tok : nullptr, no_mask ? 0 : 1, history,
        n_history, (float)rep_penalty, eos_id, suppress_eos ? 1 : 0, &samp, frame_step, skip,
        cur_stream());
    hip_check(e, "qtts_backbone_step");
    position_++;
  }

  int num_layers_, max_seq_len_, position_;
  torch::Device dev_;
  torch::Tensor embed_weight_, final_norm_weight_, codec_head_weight_, cos_table_, sin_table_, d_layer_weights_;
  std::vector<torch::Tensor> layer_weights_tensors_;
  torch::Tensor k_cache_, v_cache_, hidden_buffer_, g_normalized_, logits_, token_, ws_;
  torch::Tensor ws_streams_;   // decode_steps_streams(): per-stream workspaces
  torch::Tensor ws_shared_;    // decode_steps_streams(shared=True): the weight-shared launches' workspace
  torch::Tensor pf_ws_;        // prefill(): activations (grown on demand)
};

// ---------------------------------------------------------------------------------------
class MegakernelCodePredictorDecoder {
 public:
  MegakernelCodePredictorDecoder(std::vector<torch::Tensor> layer_weights_flat, torch::Tensor final_norm_weight,
                                 torch::Tensor cos_table, torch::Tensor sin_table, int64_t num_layers,
                                 int64_t max_seq_len)
      : num_layers_((int)num_layers), max_seq_len_((int)max_seq_len), dev_(final_norm_weight.device()) {
    TORCH_CHECK(num_layers >= 1 && max_seq_len >= 1, "num_layers and max_seq_len must be >= 1");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    check_bf16(final_norm_weight, {kHidden}, "final_norm_weight");
    TORCH_CHECK(cos_table.size(0) >= max_seq_len && sin_table.size(0) >= max_seq_len, "RoPE tables shorter than max_seq_len");
    check_bf16(cos_table, {cos_table.size(0), kHeadDim}, "cos_table");
    check_bf16(sin_table, {sin_table.size(0), kHeadDim}, "sin_table");
    final_norm_weight_ = final_norm_weight;
    cos_table_ = cos_table;
    sin_table_ = sin_table;
    layer_weights_tensors_ = layer_weights_flat;
    auto host = pack_layers(layer_weights_flat, num_layers_);
    d_layer_weights_ = upload_struct(host.data(), host.size() * sizeof(TTSLayerWeights), dev_);
    auto f32 = torch::dtype(torch::kFloat32).device(dev_);
    k_cache_ = torch::zeros({num_layers, kKVHeads, max_seq_len, kHeadDim}, f32);
    v_cache_ = torch::zeros({num_layers, kKVHeads, max_seq_len, kHeadDim}, f32);
    hidden_buffer_ = torch::zeros({kHidden}, f32);
    g_normalized_ = torch::zeros({kHidden}, f32);
    ws_ = make_workspace(dev_);
    position_ = 0;
  }
  ~MegakernelCodePredictorDecoder() {
    (void)qtts_workspace_release(ws_.data_ptr(), 1);
    if (ws_streams_.defined()) (void)qtts_workspace_release(ws_streams_.data_ptr(), kMaxStreams);
    if (ws_shared_.defined()) (void)qtts_workspace_release(ws_shared_.data_ptr(), 1);
  }
  MegakernelCodePredictorDecoder(const MegakernelCodePredictorDecoder&) = delete;
  MegakernelCodePredictorDecoder& operator=(const MegakernelCodePredictorDecoder&) = delete;

  torch::Tensor decode_step_with_embedding(torch::Tensor input_embedding) {
    TORCH_CHECK(position_ < max_seq_len_, "position ", position_, " >= max_seq_len ", max_seq_len_, " (KV cache full)");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    auto e = as_bf16_vec(input_embedding, dev_);
    hip_check(qtts_cp_step(ws_.data_ptr(), reinterpret_cast<const CPLayerWeights*>(d_layer_weights_.data_ptr()),
                           num_layers_, final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(),
                           k_cache_.data_ptr(), v_cache_.data_ptr(), max_seq_len_, position_, e.data_ptr(),
                           g_normalized_.data_ptr<float>(), hidden_buffer_.data_ptr<float>(),
                           cur_stream()),
              "qtts_cp_step");
    position_++;
    return g_normalized_.clone();
  }

  // Extended: bind the 15 lm-heads, the 15 codebook embedding tables and the backbone codec
  // embedding used by frame().
  void set_heads(std::vector<torch::Tensor> lm_heads, std::vector<torch::Tensor> embeddings, torch::Tensor bb_embedding) {
    TORCH_CHECK(!lm_heads.empty() && lm_heads.size() == embeddings.size(), "need as many lm-heads as embedding tables");
    const int64_t v = lm_heads[0].size(0);
    std::vector<const void*> hp, ep;
    for (size_t g = 0; g < lm_heads.size(); ++g) {
      check_bf16(lm_heads[g], {v, kHidden}, "lm_head");
      check_bf16(embeddings[g], {embeddings[g].size(0), kHidden}, "codec embedding");
      TORCH_CHECK(embeddings[g].size(0) >= v, "codec embedding ", g, " has fewer rows than the lm-head vocabulary");
      hp.push_back(lm_heads[g].data_ptr());
      ep.push_back(embeddings[g].data_ptr());
    }
    check_bf16(bb_embedding, {bb_embedding.size(0), kHidden}, "backbone codec embedding");
    bb_vocab_ = bb_embedding.size(0);
    heads_ = lm_heads;
    embs_ = embeddings;
    bb_emb_ = bb_embedding;
    cp_vocab_ = (int)v;
    d_heads_ = upload_struct(hp.data(), hp.size() * sizeof(void*), dev_);
    d_embs_ = upload_struct(ep.data(), ep.size() * sizeof(void*), dev_);
  }

  // Extended: one whole frame (2-token prefill + 14 decode steps + 15 heads + combine).
  void frame(torch::Tensor bb_hidden, torch::Tensor g0, c10::optional<torch::Tensor> text_row, torch::Tensor out_tokens,
             torch::Tensor out_combined, int64_t eos_id, torch::Tensor done, bool do_sample, double temperature,
             int64_t top_k, double top_p, int64_t seed, int64_t frame_step, c10::optional<torch::Tensor> history_slot) {
    TORCH_CHECK(!heads_.empty(), "call set_heads() before frame()");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    TORCH_CHECK(bb_hidden.is_cuda() && bb_hidden.scalar_type() == torch::kFloat32 && bb_hidden.numel() == kHidden &&
                    bb_hidden.is_contiguous(), "bb_hidden must be a contiguous f32 GPU tensor of 1024 values");
    TORCH_CHECK(g0.is_cuda() && g0.scalar_type() == torch::kInt32, "g0 must be an int32 GPU tensor");
    TORCH_CHECK(out_tokens.is_cuda() && out_tokens.scalar_type() == torch::kInt32 &&
                    out_tokens.numel() >= (int64_t)heads_.size() + 1, "out_tokens must be int32 GPU with >= groups+1 entries");
    TORCH_CHECK(out_combined.is_cuda() && out_combined.scalar_type() == torch::kBFloat16 && out_combined.numel() == kHidden,
                "out_combined must be a bf16 GPU tensor of 1024 values");
    TORCH_CHECK(done.is_cuda() && done.scalar_type() == torch::kInt32, "done must be an int32 GPU tensor");
    TORCH_CHECK((int)heads_.size() + 1 <= max_seq_len_, "max_seq_len too small for a frame");
    const void* tr = nullptr;
    if (text_row.has_value()) {
      TORCH_CHECK(text_row->is_cuda() && text_row->scalar_type() == torch::kBFloat16 && text_row->numel() == kHidden &&
                      text_row->is_contiguous(), "text_row must be a contiguous bf16 GPU tensor of 1024 values");
      tr = text_row->data_ptr();
    }
    int* hs = nullptr;
    if (history_slot.has_value()) {
      TORCH_CHECK(history_slot->is_cuda() && history_slot->scalar_type() == torch::kInt32 && history_slot->numel() >= 1,
                  "history_slot must be an int32 GPU tensor");
      hs = history_slot->data_ptr<int>();
    }
    QttsSampling s = sampling(do_sample, temperature, top_k, top_p, seed);
    hip_check(qtts_cp_frame(ws_.data_ptr(), reinterpret_cast<const CPLayerWeights*>(d_layer_weights_.data_ptr()),
                            num_layers_, final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(),
                            k_cache_.data_ptr(), v_cache_.data_ptr(), max_seq_len_, bb_hidden.data_ptr<float>(),
                            g0.data_ptr<int>(), bb_emb_.data_ptr(), reinterpret_cast<const void* const*>(d_heads_.data_ptr()),
                            reinterpret_cast<const void* const*>(d_embs_.data_ptr()), (int)heads_.size(), cp_vocab_, tr,
                            out_tokens.data_ptr<int>(), out_combined.data_ptr(), hs, (int)eos_id, done.data_ptr<int>(), &s,
                            (int)frame_step, cur_stream()),
              "qtts_cp_frame");
  }

  // Extended: frames of n (1..8) independent streams in one launch, stream s on XCD s (its own
  // workspace and KV cache, allocated on first use); row s of each argument belongs to stream s.
  void frames_streams(torch::Tensor bb_hidden, torch::Tensor g0, c10::optional<torch::Tensor> text_rows,
                      torch::Tensor out_tokens, torch::Tensor out_combined, int64_t eos_id, torch::Tensor done,
                      bool do_sample, double temperature, int64_t top_k, double top_p, int64_t seed, int64_t frame_step,
                      bool shared) {
    TORCH_CHECK(!heads_.empty(), "call set_heads() before frames_streams()");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    const int64_t n = bb_hidden.size(0);
    const int64_t groups = (int64_t)heads_.size();
    TORCH_CHECK(n >= 1 && n <= kMaxStreams, "1..", kMaxStreams, " streams per launch, got ", n);
    TORCH_CHECK(bb_hidden.is_cuda() && bb_hidden.scalar_type() == torch::kFloat32 && bb_hidden.dim() == 2 &&
                    bb_hidden.size(1) == kHidden && bb_hidden.is_contiguous(), "bb_hidden must be contiguous f32 [n, 1024]");
    TORCH_CHECK(g0.is_cuda() && g0.scalar_type() == torch::kInt32 && g0.numel() == n && g0.is_contiguous(), "g0 must be int32 [n]");
    TORCH_CHECK(out_tokens.is_cuda() && out_tokens.scalar_type() == torch::kInt32 && out_tokens.dim() == 2 &&
                    out_tokens.size(0) == n && out_tokens.size(1) == groups + 1 && out_tokens.is_contiguous(),
                "out_tokens must be contiguous int32 [n, groups + 1]");
    TORCH_CHECK(out_combined.is_cuda() && out_combined.scalar_type() == torch::kBFloat16 && out_combined.dim() == 2 &&
                    out_combined.size(0) == n && out_combined.size(1) == kHidden && out_combined.is_contiguous(),
                "out_combined must be contiguous bf16 [n, 1024]");
    TORCH_CHECK(done.is_cuda() && done.scalar_type() == torch::kInt32 && done.numel() == n && done.is_contiguous(), "done must be int32 [n]");
    const void* tr = nullptr;
    if (text_rows.has_value()) {
      TORCH_CHECK(text_rows->is_cuda() && text_rows->scalar_type() == torch::kBFloat16 && text_rows->dim() == 2 &&
                      text_rows->size(0) == n && text_rows->size(1) == kHidden && text_rows->is_contiguous(),
                  "text_rows must be contiguous bf16 [n, 1024]");
      tr = text_rows->data_ptr();
    }
    if (!k_streams_.defined()) {
      auto f32 = torch::dtype(torch::kFloat32).device(dev_);
      k_streams_ = torch::zeros({kMaxStreams, num_layers_, kKVHeads, max_seq_len_, kHeadDim}, f32);
      v_streams_ = torch::zeros({kMaxStreams, num_layers_, kKVHeads, max_seq_len_, kHeadDim}, f32);
    }
    QttsSampling smp = sampling(do_sample, temperature, top_k, top_p, seed);
    if (shared) {
      ensure_shared_ws(ws_shared_, dev_);
      hip_check(qtts_cp_frame_shared((int)n, ws_shared_.data_ptr(), reinterpret_cast<const CPLayerWeights*>(d_layer_weights_.data_ptr()),
                                     num_layers_, final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(),
                                     k_streams_.data_ptr(), v_streams_.data_ptr(), max_seq_len_, bb_hidden.data_ptr<float>(),
                                     g0.data_ptr<int>(), bb_emb_.data_ptr(), reinterpret_cast<const void* const*>(d_heads_.data_ptr()),
                                     reinterpret_cast<const void* const*>(d_embs_.data_ptr()), (int)groups, cp_vocab_, tr,
                                     out_tokens.data_ptr<int>(), out_combined.data_ptr(), (int)eos_id, done.data_ptr<int>(), &smp,
                                     (int)frame_step, cur_stream()),
                "qtts_cp_frame_shared");
      return;
    }
    if (!ws_streams_.defined()) {
      ws_streams_ = torch::zeros({(int64_t)(kMaxStreams * qtts_workspace_bytes())}, torch::dtype(torch::kUInt8).device(dev_));
      hip_check(qtts_workspace_init(ws_streams_.data_ptr(), dev_.index()), "qtts_workspace_init");
    }
    hip_check(qtts_cp_frame_streams((int)n, ws_streams_.data_ptr(), reinterpret_cast<const CPLayerWeights*>(d_layer_weights_.data_ptr()),
                                    num_layers_, final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(),
                                    k_streams_.data_ptr(), v_streams_.data_ptr(), max_seq_len_, bb_hidden.data_ptr<float>(),
                                    g0.data_ptr<int>(), bb_emb_.data_ptr(), reinterpret_cast<const void* const*>(d_heads_.data_ptr()),
                                    reinterpret_cast<const void* const*>(d_embs_.data_ptr()), (int)groups, cp_vocab_, tr,
                                    out_tokens.data_ptr<int>(), out_combined.data_ptr(), (int)eos_id, done.data_ptr<int>(), &smp,
                                    (int)frame_step, cur_stream()),
              "qtts_cp_frame_streams");
  }
  void check_error_streams() const {
    check_shared_error(ws_shared_);
    if (!ws_streams_.defined()) return;
    for (int st = 0; st < kMaxStreams; ++st) {
      unsigned int code = 0;
      hip_check(qtts_workspace_check(static_cast<uint8_t*>(ws_streams_.data_ptr()) + st * qtts_workspace_bytes(), &code, cur_stream()),
                "qtts_workspace_check");
      TORCH_CHECK(code == 0, "stream ", st, ": decode kernel reported a device-side wait timeout (error word ", code, ")");
    }
  }


  void reset() {
    position_ = 0;
    k_cache_.zero_();
    v_cache_.zero_();
  }
  int64_t position() const { return position_; }
  void set_position(int64_t pos) {
    TORCH_CHECK(pos >= 0 && pos <= max_seq_len_, "position ", pos, " outside [0, ", max_seq_len_, "]");
    position_ = (int)pos;
  }
  torch::Tensor get_hidden_states() const { return g_normalized_.clone(); }
  torch::Tensor get_k_cache() const { return k_cache_; }
  torch::Tensor get_v_cache() const { return v_cache_; }
  void check_error() const { check_device_error(ws_); }
  // test hook: pre-sets the workspace's error word (after at least one launch), so that every
  // wait of the next launch gives up at its first check
  void debug_set_error(int64_t code) {
    hip_check(qtts_debug_set_error(ws_.data_ptr(), (unsigned int)code, cur_stream()), "qtts_debug_set_error");
  }

  void set_kv_cache(torch::Tensor k_cache, torch::Tensor v_cache) {
    TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes(), "k/v must be [layers, 8, seq, 128]");
    TORCH_CHECK(k_cache.size(0) == num_layers_ && k_cache.size(1) == kKVHeads && k_cache.size(3) == kHeadDim,
                "k/v must be [", num_layers_, ", 8, seq, 128], got ", k_cache.sizes());
    TORCH_CHECK(k_cache.size(2) <= max_seq_len_, "k/v longer than max_seq_len");
    using namespace torch::indexing;
    k_cache_.index_put_({Slice(), Slice(), Slice(0, k_cache.size(2)), Slice()}, k_cache.to(dev_, torch::kFloat32));
    v_cache_.index_put_({Slice(), Slice(), Slice(0, v_cache.size(2)), Slice()}, v_cache.to(dev_, torch::kFloat32));
  }

 private:
  int num_layers_, max_seq_len_, position_, cp_vocab_ = 0;
  int64_t bb_vocab_ = 0;
  torch::Device dev_;
  torch::Tensor final_norm_weight_, cos_table_, sin_table_, d_layer_weights_;
  std::vector<torch::Tensor> layer_weights_tensors_, heads_, embs_;
  torch::Tensor bb_emb_, d_heads_, d_embs_;
  torch::Tensor k_cache_, v_cache_, hidden_buffer_, g_normalized_, ws_;
  torch::Tensor ws_streams_, k_streams_, v_streams_;   // frames_streams(): per-stream workspaces and KV caches
  torch::Tensor ws_shared_;                            // frames_streams(shared=True): the weight-shared launches' workspace
};

// ---------------------------------------------------------------------------------------
// Paged-cache operators: functions over tensors (no reference counterpart).
using torch::Tensor;
using OptTensor = c10::optional<torch::Tensor>;

const int* check_i32(const Tensor& t, const torch::Device& dev, int64_t n, const char* name) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev, ", got ", t.device());
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.is_contiguous(), name, " must be a contiguous int32 tensor");
  TORCH_CHECK(t.numel() >= n, name, " needs ", n, " entries, got ", t.numel());
  return t.data_ptr<int>();
}

void check_aligned(const Tensor& t, const char* name) {
  TORCH_CHECK((reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0, name, " must be 16-byte aligned");
}

// block_table [requests, width] int32, rows of its own stride
void check_table(const Tensor& t, const torch::Device& dev, int64_t requests) {
  TORCH_CHECK(t.device() == dev, "block_table must be on ", dev, ", got ", t.device());
  TORCH_CHECK(t.scalar_type() == torch::kInt32 && t.dim() == 2 && t.size(0) >= requests && t.size(1) >= 1,
              "block_table must be an int32 [requests, width] tensor with >= ", requests, " rows");
  TORCH_CHECK(t.stride(1) == 1 || t.size(1) == 1, "block_table rows must be contiguous");
  TORCH_CHECK(t.size(0) == 1 || t.stride(0) >= t.size(1), "block_table rows must not overlap");
}
void check_capacity(const Tensor& t, int64_t page_size) {
  TORCH_CHECK(t.size(1) <= (1ll << 30) / page_size, "a block_table row holds more than 2^30 tokens");
}
long long table_stride(const Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

void check_page_size(int64_t page_size, int64_t least) {
  TORCH_CHECK(page_size >= least && page_size <= 65536 && (page_size & (page_size - 1)) == 0,
              "page_size must be a power of two in [", least, ", 65536], got ", page_size);
}

QttsPagedCache paged_cache(const Tensor& k, const Tensor& v) {
  TORCH_CHECK(k.is_cuda(), "k_cache must be a GPU tensor");
  TORCH_CHECK(k.scalar_type() == torch::kBFloat16 || k.scalar_type() == torch::kFloat16,
              "the cache must be bfloat16 or float16, got ", k.scalar_type());
  TORCH_CHECK(k.dim() == 4, "k_cache must be [pages, kv_heads, page_size, head_dim], got ", k.sizes());
  TORCH_CHECK(v.device() == k.device() && v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes() && v.strides() == k.strides(),
              "v_cache must be like k_cache (device, type, shape and strides)");
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, "head_dim must be 64 or 128, got ", k.size(3));
  check_page_size(k.size(2), 16);
  TORCH_CHECK(k.size(0) >= 1 && k.size(0) <= INT_MAX && k.size(1) >= 1 && k.size(1) <= INT_MAX, "empty cache: ", k.sizes());
  TORCH_CHECK(k.stride(3) == 1, "the cache's channels must be contiguous");
  for (int i = 0; i < 3; ++i) TORCH_CHECK(k.stride(i) >= 0 && k.stride(i) % 8 == 0, "cache strides must be multiples of 8, got ", k.strides());
  TORCH_CHECK(k.stride(2) >= k.size(3) && k.stride(2) <= (1 << 24) && k.stride(1) <= INT_MAX && k.stride(0) <= INT_MAX, "cache strides out of range: ", k.strides());
  check_aligned(k, "k_cache");
  check_aligned(v, "v_cache");
  QttsPagedCache c;
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.dtype = k.scalar_type() == torch::kBFloat16 ? QTTS_BF16 : QTTS_F16;
  c.num_pages = (int)k.size(0);
  c.num_kv_heads = (int)k.size(1);
  c.page_size = (int)k.size(2);
  c.head_dim = (int)k.size(3);
  c.page_stride = k.stride(0);
  c.head_stride = k.stride(1);
  c.slot_stride = k.stride(2);
  return c;
}

// [tokens, heads, head_dim] of the cache's type; channels contiguous, the other strides multiples of 8
void check_heads(const Tensor& t, const Tensor& cache, int64_t tokens, int64_t heads, const char* name) {
  TORCH_CHECK(t.device() == cache.device(), name, " must be on ", cache.device(), ", got ", t.device());
  TORCH_CHECK(t.scalar_type() == cache.scalar_type(), name, " must be of the cache's type ", cache.scalar_type(), ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 3 && t.size(0) == tokens && (heads < 0 || t.size(1) == heads) && t.size(1) >= 1 && t.size(2) == cache.size(3),
              name, " must be [", tokens, ", ", heads < 0 ? std::string("heads") : std::to_string(heads), ", ", cache.size(3), "], got ", t.sizes());
  if (t.numel() == 0) return;
  TORCH_CHECK(t.stride(2) == 1, name, ": channels must be contiguous");
  TORCH_CHECK((t.size(0) == 1 || t.stride(0) % 8 == 0) && (t.size(1) == 1 || t.stride(1) % 8 == 0), name,
              ": token and head strides must be multiples of 8, got ", t.strides());
  check_aligned(t, name);
}
long long tok_stride(const Tensor& t) { return t.size(0) == 1 ? 0 : t.stride(0); }
long long head_stride(const Tensor& t) { return t.size(1) == 1 ? 0 : t.stride(1); }

std::vector<Tensor> paged_plan(Tensor new_tokens, Tensor lengths, Tensor block_table, Tensor free_pages, Tensor free_count,
                               int64_t page_size, int64_t total_tokens, OptTensor lengths_out, OptTensor free_count_out) {
  TORCH_CHECK(new_tokens.is_cuda(), "new_tokens must be a GPU tensor");
  const torch::Device dev = new_tokens.device();
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  const int64_t n = new_tokens.numel();
  TORCH_CHECK(n >= 1 && n <= (1 << 24), "a plan takes 1 .. 2^24 requests, got ", n);
  TORCH_CHECK(total_tokens >= 0 && total_tokens <= (1 << 30), "total_tokens out of range: ", total_tokens);
  const int* nt = check_i32(new_tokens, dev, n, "new_tokens");
  int* len = const_cast<int*>(check_i32(lengths, dev, n, "lengths"));
  check_table(block_table, dev, n);
  const int* fp = check_i32(free_pages, dev, 0, "free_pages");
  int* fc = const_cast<int*>(check_i32(free_count, dev, 1, "free_count"));
  check_page_size(page_size, 1);
  check_capacity(block_table, page_size);
  int* len_out = lengths_out.has_value() ? const_cast<int*>(check_i32(*lengths_out, dev, n, "lengths_out")) : len;
  int* fc_out = free_count_out.has_value() ? const_cast<int*>(check_i32(*free_count_out, dev, 1, "free_count_out")) : fc;
  auto parts = torch::empty({2 * total_tokens + 3 * n + 1}, torch::dtype(torch::kInt32).device(dev))
                   .split_with_sizes({total_tokens, total_tokens, n + 1, n, n});
  auto &slots = parts[0], &positions = parts[1], &cu = parts[2], &kv = parts[3], &status = parts[4];
  hip_check(qtts_paged_plan((int)n, (int)block_table.size(1), table_stride(block_table), (int)page_size, (int)total_tokens, nt, len,
                            block_table.data_ptr<int>(), fp, (int)std::min<int64_t>(free_pages.numel(), INT_MAX), fc,
                            slots.data_ptr<int>(), positions.data_ptr<int>(), cu.data_ptr<int>(), kv.data_ptr<int>(), len_out,
                            fc_out, status.data_ptr<int>(), cur_stream()),
            "qtts_paged_plan");
  return parts;
}

void paged_release(Tensor release, Tensor lengths, Tensor block_table, Tensor free_pages, Tensor free_count, int64_t page_size) {
  TORCH_CHECK(release.is_cuda(), "release must be a GPU tensor");
  const torch::Device dev = release.device();
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  const int64_t n = release.numel();
  TORCH_CHECK(n >= 1 && n <= (1 << 24), "a release takes 1 .. 2^24 requests, got ", n);
  const int* rel = check_i32(release, dev, n, "release");
  check_i32(lengths, dev, n, "lengths");
  check_table(block_table, dev, n);
  check_i32(free_pages, dev, 1, "free_pages");
  check_i32(free_count, dev, 1, "free_count");
  check_page_size(page_size, 1);
  hip_check(qtts_paged_release((int)n, (int)block_table.size(1), table_stride(block_table), (int)page_size, rel,
                               lengths.data_ptr<int>(), block_table.data_ptr<int>(), free_pages.data_ptr<int>(),
                               (int)std::min<int64_t>(free_pages.numel(), INT_MAX), free_count.data_ptr<int>(), cur_stream()),
            "qtts_paged_release");
}

Tensor qk_norm_rope_store(Tensor q, Tensor k, Tensor v, OptTensor q_weight, OptTensor k_weight, Tensor cos_table, Tensor sin_table,
                          Tensor positions, Tensor slots, Tensor k_cache, Tensor v_cache, double eps,
                          std::vector<int64_t> mrope_section, OptTensor out) {
  const QttsPagedCache cache = paged_cache(k_cache, v_cache);
  const torch::Device dev = k_cache.device();
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  const int64_t n = q.dim() == 3 ? q.size(0) : -1, dim = cache.head_dim;
  TORCH_CHECK(n >= 0 && n <= INT_MAX, "q must be [tokens, heads, head_dim], got ", q.sizes());
  check_heads(q, k_cache, n, -1, "q");
  check_heads(k, k_cache, n, cache.num_kv_heads, "k");
  check_heads(v, k_cache, n, cache.num_kv_heads, "v");
  TORCH_CHECK(q.size(1) <= INT_MAX, "too many heads");
  for (const OptTensor* w : {&q_weight, &k_weight})
    if (w->has_value()) {
      TORCH_CHECK((*w)->device() == dev && (*w)->scalar_type() == k_cache.scalar_type() && (*w)->is_contiguous() && (*w)->dim() == 1 &&
                      (*w)->size(0) == dim, "norm weights must be contiguous [", dim, "] tensors of the cache's type on ", dev);
      check_aligned(**w, "norm weights");
    }
  TORCH_CHECK(cos_table.device() == dev && cos_table.dim() == 2 && cos_table.size(0) >= 1 && cos_table.size(0) <= INT_MAX &&
                  cos_table.size(1) == dim && cos_table.is_contiguous(), "cos must be a contiguous [rows, ", dim, "] tensor on ", dev);
  TORCH_CHECK(cos_table.scalar_type() == k_cache.scalar_type() || cos_table.scalar_type() == torch::kFloat32,
              "cos and sin must be of the cache's type or float32");
  TORCH_CHECK(sin_table.device() == dev && sin_table.scalar_type() == cos_table.scalar_type() && sin_table.sizes() == cos_table.sizes() &&
                  sin_table.is_contiguous(), "sin must be like cos");
  check_aligned(cos_table, "cos");
  check_aligned(sin_table, "sin");
  const bool three = positions.dim() == 2;
  TORCH_CHECK((positions.dim() == 1 && positions.size(0) == n) || (three && positions.size(0) == 3 && positions.size(1) == n),
              "positions must be [", n, "] or [3, ", n, "], got ", positions.sizes());
  const int* pos = check_i32(positions, dev, n, "positions");
  const int* slot = check_i32(slots, dev, n, "slots");
  TORCH_CHECK(slots.numel() == n, "slots must have one entry per token");
  int64_t h = 0, w = 0;
  if (three) {
    TORCH_CHECK(mrope_section.size() == 3 && mrope_section[0] >= 0 && mrope_section[1] >= 0 && mrope_section[2] >= 0 &&
                    mrope_section[0] + mrope_section[1] + mrope_section[2] == dim / 2,
                "mrope_section must be three counts that add up to head_dim / 2 = ", dim / 2);
    h = 3 * mrope_section[1];
    w = 3 * mrope_section[2];
    TORCH_CHECK(h <= dim / 2 && w <= dim / 2, "mrope_section: h and w take at most a third of the channels each");
  }
  TORCH_CHECK(eps >= 0.0, "eps must be >= 0");
  Tensor o;
  if (out.has_value()) {
    o = *out;
    check_heads(o, k_cache, n, q.size(1), "out");
    at::assert_no_internal_overlap(o);
  } else {
    o = torch::empty({n, q.size(1), dim}, q.options());
  }
  if (n == 0) return o;
  at::assert_no_internal_overlap(k_cache);   // (an expanded cache: its rows are one)
  at::assert_no_internal_overlap(v_cache);
  hip_check(qtts_qk_norm_rope_store(&cache, (int)n, (int)q.size(1), q.data_ptr(), tok_stride(q), head_stride(q), k.data_ptr(),
                                    tok_stride(k), head_stride(k), v.data_ptr(), tok_stride(v), head_stride(v), o.data_ptr(),
                                    tok_stride(o), head_stride(o), q_weight.has_value() ? q_weight->data_ptr() : nullptr,
                                    k_weight.has_value() ? k_weight->data_ptr() : nullptr, (float)eps, cos_table.data_ptr(),
                                    sin_table.data_ptr(), cos_table.scalar_type() == torch::kFloat32, (int)cos_table.size(0), pos,
                                    three ? n : 0, (int)h, (int)w, slot, cur_stream()),
            "qtts_qk_norm_rope_store");
  return o;
}

// what both attention calls check: returns the output tensor
Tensor check_attention(const QttsPagedCache& cache, const Tensor& q, const Tensor& k_cache, const Tensor& block_table,
                       const Tensor& kv_lens, int64_t requests, double scale, int64_t window, int64_t sinks, OptTensor out) {
  const torch::Device dev = k_cache.device();
  TORCH_CHECK(q.dim() == 3, "q must be [tokens, heads, head_dim], got ", q.sizes());
  check_heads(q, k_cache, q.size(0), -1, "q");
  TORCH_CHECK(q.size(1) % cache.num_kv_heads == 0, "q's heads (", q.size(1), ") must be a multiple of the cache's (", cache.num_kv_heads, ")");
  TORCH_CHECK(q.size(0) * q.size(1) <= INT_MAX / 2, "q has too many rows");
  TORCH_CHECK(requests >= 1 && requests <= INT_MAX, "at least one request is needed");
  check_table(block_table, dev, requests);
  check_capacity(block_table, cache.page_size);
  check_i32(kv_lens, dev, requests, "kv_lens");
  TORCH_CHECK(scale > 0.0 && std::isfinite((float)scale) && (float)scale > 0.0f, "scale must be positive and finite");
  TORCH_CHECK(window >= 0 && window <= INT_MAX && sinks >= 0 && sinks <= INT_MAX, "window and sinks must be >= 0");
  if (!out.has_value()) return torch::empty({q.size(0), q.size(1), q.size(2)}, q.options());
  check_heads(*out, k_cache, q.size(0), q.size(1), "out");
  at::assert_no_internal_overlap(*out);
  return *out;
}

Tensor paged_attention_decode(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor kv_lens, double scale,
                              int64_t window, int64_t sinks, int64_t max_len, OptTensor out) {
  const QttsPagedCache cache = paged_cache(k_cache, v_cache);
  const torch::Device dev = k_cache.device();
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  const int64_t n = q.dim() == 3 ? q.size(0) : 0;
  Tensor o = check_attention(cache, q, k_cache, block_table, kv_lens, n, scale, window, sinks, out);
  const int width = (int)block_table.size(1);
  TORCH_CHECK(max_len >= 1, "max_len must be >= 1");
  const int most = (int)std::min<int64_t>(max_len, (int64_t)width * cache.page_size);
  const size_t need = qtts_paged_decode_workspace_bytes((int)n, (int)q.size(1), cache.num_kv_heads, cache.head_dim, width,
                                                        cache.page_size, most, (int)window, (int)sinks);
  Tensor ws;
  if (need > 0) ws = torch::empty({(int64_t)need}, torch::dtype(torch::kUInt8).device(dev));
  hip_check(qtts_paged_attention_decode(&cache, (int)n, (int)q.size(1), q.data_ptr(), tok_stride(q), head_stride(q), o.data_ptr(),
                                        tok_stride(o), head_stride(o), block_table.data_ptr<int>(), width, table_stride(block_table),
                                        kv_lens.data_ptr<int>(), most, (float)scale, (int)window, (int)sinks,
                                        need > 0 ? ws.data_ptr() : nullptr, need, cur_stream()),
            "qtts_paged_attention_decode");
  return o;
}

Tensor paged_attention_prefill(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, Tensor kv_lens, Tensor cu_tokens,
                               double scale, int64_t window, int64_t sinks, int64_t max_len, OptTensor out) {
  const QttsPagedCache cache = paged_cache(k_cache, v_cache);
  const torch::Device dev = k_cache.device();
  c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  TORCH_CHECK(max_len >= 1, "max_len must be >= 1");
  const int64_t n = cu_tokens.numel() - 1;
  Tensor o = check_attention(cache, q, k_cache, block_table, kv_lens, n, scale, window, sinks, out);
  const int* cu = check_i32(cu_tokens, dev, n + 1, "cu_tokens");
  if (q.size(0) == 0) return o;
  hip_check(qtts_paged_attention_prefill(&cache, (int)n, (int)q.size(0), (int)q.size(1), q.data_ptr(), tok_stride(q), head_stride(q),
                                         o.data_ptr(), tok_stride(o), head_stride(o), block_table.data_ptr<int>(),
                                         (int)block_table.size(1), table_stride(block_table), kv_lens.data_ptr<int>(), cu,
                                         (int)std::min<int64_t>(max_len, INT_MAX), (float)scale, (int)window, (int)sinks, cur_stream()),
            "qtts_paged_attention_prefill");
  return o;
}

// The backbone over a paged cache for any number of streams: weights, and one call per packed batch of new tokens.
class PagedTTSBackbone {
 public:
  PagedTTSBackbone(std::vector<Tensor> layer_weights_flat, Tensor final_norm_weight, Tensor codec_head_weight, Tensor cos_table,
                   Tensor sin_table, int64_t num_layers)
      : num_layers_((int)num_layers), dev_(final_norm_weight.device()) {
    TORCH_CHECK(num_layers >= 1, "num_layers must be >= 1");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    TORCH_CHECK(codec_head_weight.dim() == 2, "codec_head_weight must be [vocab, 1024]");
    check_bf16(codec_head_weight, {codec_head_weight.size(0), kHidden}, "codec_head_weight");
    check_bf16(final_norm_weight, {kHidden}, "final_norm_weight");
    TORCH_CHECK(cos_table.dim() == 2 && cos_table.size(0) >= 1 && sin_table.sizes() == cos_table.sizes(), "RoPE tables must be alike");
    check_bf16(cos_table, {cos_table.size(0), kHeadDim}, "cos_table");
    check_bf16(sin_table, {sin_table.size(0), kHeadDim}, "sin_table");
    final_norm_weight_ = final_norm_weight;
    codec_head_weight_ = codec_head_weight;
    cos_table_ = cos_table;
    sin_table_ = sin_table;
    layers_ = layer_weights_flat;
    host_ = pack_layers(layer_weights_flat, num_layers_);
    table_ = upload_struct(host_.data(), host_.size() * sizeof(TTSLayerWeights), dev_);
  }

  // embeds bf16 [tokens, 1024]; k_pool, v_pool bf16 [layers, pages, 8, page_size, 128]; the plan's tensors (cu_tokens
  // None: one token for each of kv_lens' streams). Returns the hiddens f32 [streams, 1024]; with out_tokens every stream's
  // token is selected. history int32 [streams, H] with n_history: an int for all or an int32 tensor [streams].
  Tensor forward(Tensor embeds, Tensor k_pool, Tensor v_pool, Tensor block_table, Tensor slots, Tensor positions, OptTensor cu_tokens,
                 Tensor kv_lens, int64_t max_len, int64_t window, int64_t sinks, OptTensor out_tokens, OptTensor history,
                 OptTensor n_history, int64_t history_len, double repetition_penalty, int64_t eos_id, bool suppress_eos,
                 bool do_sample, double temperature, int64_t top_k, double top_p, int64_t seed, int64_t frame_step, OptTensor skip,
                 OptTensor out_logits) {
    c10::hip::HIPGuardMasqueradingAsCUDA guard(dev_);
    TORCH_CHECK(k_pool.dim() == 5 && k_pool.size(0) == num_layers_ && v_pool.sizes() == k_pool.sizes() && v_pool.strides() == k_pool.strides(),
                "k_pool and v_pool must be [", num_layers_, ", pages, 8, page_size, 128], got ", k_pool.sizes());
    const QttsPagedCache cache = paged_cache(k_pool.select(0, 0), v_pool.select(0, 0));
    TORCH_CHECK(k_pool.device() == dev_ && cache.dtype == QTTS_BF16 && cache.num_kv_heads == kKVHeads && cache.head_dim == kHeadDim,
                "the pool must be bfloat16 with 8 heads of 128 on ", dev_);
    TORCH_CHECK(k_pool.stride(0) % 8 == 0, "pool strides must be multiples of 8");
    const int64_t n = kv_lens.numel(), tokens = embeds.size(0);
    TORCH_CHECK(n >= 1 && n <= 65535, "1 .. 65535 streams, got ", n);
    check_bf16(embeds, {tokens, kHidden}, "embeds");
    TORCH_CHECK(embeds.device() == dev_ && tokens >= 1 && tokens <= (1 << 20), "embeds must be [1 .. 2^20, 1024] on ", dev_);
    check_aligned(embeds, "embeds");
    TORCH_CHECK(cu_tokens.has_value() || tokens == n, "one token for each stream expected (", n, "), got ", tokens);
    check_table(block_table, dev_, n);
    check_capacity(block_table, cache.page_size);
    const int width = (int)block_table.size(1);
    TORCH_CHECK(max_len >= 1 && window >= 0 && window <= INT_MAX && sinks >= 0 && sinks <= INT_MAX, "max_len, window or sinks out of range");
    const int most = (int)std::min<int64_t>(max_len, (int64_t)width * cache.page_size);
    int* tok = nullptr;
    if (out_tokens.has_value()) tok = const_cast<int*>(check_i32(*out_tokens, dev_, n, "out_tokens"));
    const int* hist = nullptr;
    int hstride = 0;
    if (history.has_value()) {
      hist = check_i32(*history, dev_, 0, "history");
      TORCH_CHECK(history->dim() == 2 && history->size(0) >= n, "history must be [streams, H]");
      hstride = (int)history->size(1);
      TORCH_CHECK(history_len >= 0 && history_len <= hstride, "n_history = ", history_len, " outside [0, ", hstride, "]");
    }
    const int vocab = (int)codec_head_weight_.size(0);
    float* logits = nullptr;
    if (out_logits.has_value()) {
      TORCH_CHECK(tok != nullptr, "out_logits needs out_tokens");
      TORCH_CHECK(out_logits->device() == dev_ && out_logits->scalar_type() == torch::kFloat32 && out_logits->is_contiguous() &&
                      out_logits->dim() == 2 && out_logits->size(0) == n && out_logits->size(1) == vocab,
                  "out_logits must be a contiguous f32 [", n, ", ", vocab, "] tensor on ", dev_);
      logits = out_logits->data_ptr<float>();
    }
    const size_t need = qtts_paged_workspace_bytes((int)tokens, (int)n, tok ? vocab : 0, width, cache.page_size, most, (int)window, (int)sinks);
    TORCH_CHECK(need > 0, "paged workspace size query failed");
    Tensor ws = torch::empty({(int64_t)need}, torch::dtype(torch::kUInt8).device(dev_));
    Tensor hidden = torch::empty({n, kHidden}, torch::dtype(torch::kFloat32).device(dev_));
    QttsSampling samp = sampling(do_sample, temperature, top_k, top_p, seed);
    hip_check(qtts_backbone_paged(ws.data_ptr(), need, reinterpret_cast<const TTSLayerWeights*>(table_.data_ptr()), host_.data(), num_layers_,
                                  final_norm_weight_.data_ptr(), cos_table_.data_ptr(), sin_table_.data_ptr(), (int)cos_table_.size(0),
                                  &cache, k_pool.stride(0), (int)n, (int)tokens, check_i32(slots, dev_, tokens, "slots"),
                                  check_i32(positions, dev_, tokens, "positions"),
                                  cu_tokens.has_value() ? check_i32(*cu_tokens, dev_, n + 1, "cu_tokens") : nullptr,
                                  check_i32(kv_lens, dev_, n, "kv_lens"), block_table.data_ptr<int>(), width, table_stride(block_table), most,
                                  (int)window, (int)sinks, embeds.data_ptr(), hidden.data_ptr<float>(),
                                  tok ? codec_head_weight_.data_ptr() : nullptr, vocab, logits, tok, 1, hist, hstride,
                                  n_history.has_value() ? check_i32(*n_history, dev_, n, "n_history") : nullptr, (int)history_len,
                                  (float)repetition_penalty, (int)eos_id, suppress_eos ? 1 : 0, &samp, (int)frame_step,
                                  skip.has_value() ? check_i32(*skip, dev_, n, "skip") : nullptr, cur_stream()),
              "qtts_backbone_paged");
    return hidden;
  }

 private:
  int num_layers_;
  torch::Device dev_;
  std::vector<TTSLayerWeights> host_;
  std::vector<Tensor> layers_;
  Tensor final_norm_weight_, codec_head_weight_, cos_table_, sin_table_, table_;
};

}  // namespace

PYBIND11_MODULE(_qwentts_amd_C, m) {
  m.doc() = "MI355X decode kernels for Qwen3-TTS (backbone + code predictor)";
  m.def("workspace_bytes", []() { return (int64_t)qtts_workspace_bytes(); });
  m.def("shutdown", []() { hip_check(qtts_shutdown(), "qtts_shutdown"); },
        "Free the library-owned workspaces (synchronises their devices); registered with atexit by the loader.");
  m.def("set_trace", [](c10::optional<torch::Tensor> buf) {
    if (!buf.has_value()) { hip_check(qtts_debug_trace(nullptr, 0), "qtts_debug_trace"); return; }
    TORCH_CHECK(buf->is_cuda() && buf->is_contiguous(), "trace buffer must be a contiguous GPU tensor");
    hip_check(qtts_debug_trace(buf->data_ptr(), (size_t)buf->numel() * buf->element_size()), "qtts_debug_trace");
  }, py::arg("buffer") = py::none());
  m.def("set_trace_shared", [](c10::optional<torch::Tensor> buf) {
    if (!buf.has_value()) { hip_check(qtts_debug_trace_shared(nullptr, 0), "qtts_debug_trace_shared"); return; }
    TORCH_CHECK(buf->is_cuda() && buf->is_contiguous(), "trace buffer must be a contiguous GPU tensor");
    hip_check(qtts_debug_trace_shared(buf->data_ptr(), (size_t)buf->numel() * buf->element_size()), "qtts_debug_trace_shared");
  }, py::arg("buffer") = py::none());
  m.def("paged_plan", &paged_plan, py::arg("new_tokens"), py::arg("lengths"), py::arg("block_table"), py::arg("free_pages"),
        py::arg("free_count"), py::arg("page_size"), py::arg("total_tokens"), py::arg("lengths_out") = py::none(),
        py::arg("free_count_out") = py::none());
  m.def("paged_release", &paged_release, py::arg("release"), py::arg("lengths"), py::arg("block_table"), py::arg("free_pages"),
        py::arg("free_count"), py::arg("page_size"));
  m.def("qk_norm_rope_store", &qk_norm_rope_store, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("q_weight"), py::arg("k_weight"),
        py::arg("cos"), py::arg("sin"), py::arg("positions"), py::arg("slots"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("eps"), py::arg("mrope_section"), py::arg("out") = py::none());
  m.def("paged_attention_decode", &paged_attention_decode, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("kv_lens"), py::arg("scale"), py::arg("window"), py::arg("sinks"), py::arg("max_len"),
        py::arg("out") = py::none());
  m.def("paged_attention_prefill", &paged_attention_prefill, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("kv_lens"), py::arg("cu_tokens"), py::arg("scale"), py::arg("window"), py::arg("sinks"),
        py::arg("max_len"), py::arg("out") = py::none());
  py::class_<PagedTTSBackbone>(m, "PagedTTSBackbone")
      .def(py::init<std::vector<Tensor>, Tensor, Tensor, Tensor, Tensor, int64_t>())
      .def("forward", &PagedTTSBackbone::forward, py::arg("embeds"), py::arg("k_pool"), py::arg("v_pool"), py::arg("block_table"),
           py::arg("slots"), py::arg("positions"), py::arg("cu_tokens"), py::arg("kv_lens"), py::arg("max_len"), py::arg("window") = 0,
           py::arg("sinks") = 0, py::arg("out_tokens") = py::none(), py::arg("history") = py::none(), py::arg("n_history") = py::none(),
           py::arg("history_len") = 0, py::arg("repetition_penalty") = 1.0, py::arg("eos_id") = -1, py::arg("suppress_eos") = false,
           py::arg("do_sample") = false, py::arg("temperature") = 1.0, py::arg("top_k") = 0, py::arg("top_p") = 1.0,
           py::arg("seed") = 0, py::arg("frame_step") = 0, py::arg("skip") = py::none(), py::arg("out_logits") = py::none());
  py::class_<MegakernelTTSDecoder>(m, "MegakernelTTSDecoder")
      .def(py::init<torch::Tensor, std::vector<torch::Tensor>, torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor,
                    int64_t, int64_t>())
      .def("decode_step", &MegakernelTTSDecoder::decode_step)
      .def("decode_step_with_argmax", &MegakernelTTSDecoder::decode_step_with_argmax)
      .def("decode_step_with_embedding", &MegakernelTTSDecoder::decode_step_with_embedding)
      .def("decode_step_3d", &MegakernelTTSDecoder::decode_step_3d)
      .def("decode_step_select", &MegakernelTTSDecoder::decode_step_select, py::arg("input_embedding"),
           py::arg("out_token"), py::arg("history"), py::arg("n_history"), py::arg("repetition_penalty"),
           py::arg("eos_id"), py::arg("suppress_eos"), py::arg("do_sample"), py::arg("temperature"), py::arg("top_k"),
           py::arg("top_p"), py::arg("seed"), py::arg("frame_step"), py::arg("pos3") = py::none(),
           py::arg("skip_if") = py::none())
      .def("reset", &MegakernelTTSDecoder::reset)
      .def("position", &MegakernelTTSDecoder::position)
      .def("set_position", &MegakernelTTSDecoder::set_position)
      .def("get_hidden_states", &MegakernelTTSDecoder::get_hidden_states)
      .def("get_k_cache", &MegakernelTTSDecoder::get_k_cache)
      .def("get_v_cache", &MegakernelTTSDecoder::get_v_cache)
      .def("set_kv_cache", &MegakernelTTSDecoder::set_kv_cache)
      .def("hidden_state_buffer", &MegakernelTTSDecoder::hidden_state_buffer)
      .def("residual_buffer", &MegakernelTTSDecoder::residual_buffer)
      .def("logits_buffer", &MegakernelTTSDecoder::logits_buffer)
      .def("prefill", &MegakernelTTSDecoder::prefill, py::arg("embeds"), py::arg("out_token") = py::none(),
           py::arg("eos_id") = -1, py::arg("suppress_eos") = false, py::arg("do_sample") = false,
           py::arg("temperature") = 1.0, py::arg("top_k") = 0, py::arg("top_p") = 1.0, py::arg("seed") = 0,
           py::arg("pos3") = py::none())
      .def("decode_steps_streams", &MegakernelTTSDecoder::decode_steps_streams, py::arg("decoders"), py::arg("embeds"),
           py::arg("out_tokens"), py::arg("hidden_out"), py::arg("history"), py::arg("n_history"),
           py::arg("repetition_penalty"), py::arg("eos_id"), py::arg("suppress_eos"), py::arg("do_sample"),
           py::arg("temperature"), py::arg("top_k"), py::arg("top_p"), py::arg("seed"), py::arg("frame_step"),
           py::arg("skip") = py::none(), py::arg("shared") = false)
      .def("check_error_streams", &MegakernelTTSDecoder::check_error_streams)
      .def("debug_set_error", &MegakernelTTSDecoder::debug_set_error)
      .def("check_error", &MegakernelTTSDecoder::check_error);
  py::class_<MegakernelCodePredictorDecoder>(m, "MegakernelCodePredictorDecoder")
      .def(py::init<std::vector<torch::Tensor>, torch::Tensor, torch::Tensor, torch::Tensor, int64_t, int64_t>())
      .def("decode_step_with_embedding", &MegakernelCodePredictorDecoder::decode_step_with_embedding)
      .def("set_heads", &MegakernelCodePredictorDecoder::set_heads)
      .def("frames_streams", &MegakernelCodePredictorDecoder::frames_streams, py::arg("bb_hidden"), py::arg("g0"),
           py::arg("text_rows"), py::arg("out_tokens"), py::arg("out_combined"), py::arg("eos_id"), py::arg("done"),
           py::arg("do_sample"), py::arg("temperature"), py::arg("top_k"), py::arg("top_p"), py::arg("seed"),
           py::arg("frame_step"), py::arg("shared") = false)
      .def("check_error_streams", &MegakernelCodePredictorDecoder::check_error_streams)
      .def("frame", &MegakernelCodePredictorDecoder::frame, py::arg("bb_hidden"), py::arg("g0"), py::arg("text_row"),
           py::arg("out_tokens"), py::arg("out_combined"), py::arg("eos_id"), py::arg("done"), py::arg("do_sample"),
           py::arg("temperature"), py::arg("top_k"), py::arg("top_p"), py::arg("seed"), py::arg("frame_step"),
           py::arg("history_slot") = py::none())
      .def("reset", &MegakernelCodePredictorDecoder::reset)
      .def("position", &MegakernelCodePredictorDecoder::position)
      .def("set_position", &MegakernelCodePredictorDecoder::set_position)
      .def("get_hidden_states", &MegakernelCodePredictorDecoder::get_hidden_states)
      .def("get_k_cache", &MegakernelCodePredictorDecoder::get_k_cache)
      .def("get_v_cache", &MegakernelCodePredictorDecoder::get_v_cache)
      .def("set_kv_cache", &MegakernelCodePredictorDecoder::set_kv_cache)
      .def("debug_set_error", &MegakernelCodePredictorDecoder::debug_set_error)
      .def("check_error", &MegakernelCodePredictorDecoder::check_error);
}
