// Host mirror of the layers of token models: EmbeddingLayer, DropoutLayer and GroupNormLayer (the reference's embedding
// and dropout layers are host loops).  Group norm takes its statistics over all positions of a sample, so one group of [batch,
// channels] is a layer norm; of [batch, tokens, channels] it is not one per token, which
// vtlb_groupnorm_fwd_f32 gives for batch * tokens samples of one position.
#include <cmath>
#include <cstring>

#include "vtl_host.hpp"

namespace vtl {
namespace {

size_t count(const std::vector<int>& shape) {
  size_t n = 1;
  for (int d : shape) n *= (size_t)d;
  return n;
}

struct EmbeddingGate : Gate {
  VarPtr weight;
  std::shared_ptr<DeviceBuf> ids;
  size_t n;
  float scale;
  DropoutLayer::Mask mask;
  // parents: the tokens, which have no gradient, and the table
  std::vector<Tensor> backward(const Tensor& g) override {
    if (!weight->requires_grad) return {Tensor(), Tensor()};
    Session* s = g.session();
    const auto& ws = weight->value.shape();
    Tensor dW = Tensor::empty(s, ws);
    s->check(vtlb_embedding_bwd_f32(s->ctx, g.data(), ids->ptr, n, ws[0], ws[1], scale, mask.p, mask.seed, mask.step,
                                    dW.data(), 0));
    if (s->comm_on) s->check(vtlb_allreduce_sum_f32_async(s->ctx, dW.data(), dW.size()));
    return {Tensor(), dW};
  }
};

struct DropoutGate : Gate {
  DropoutLayer::Mask mask;
  std::vector<Tensor> backward(const Tensor& g) override {
    Session* s = g.session();
    Tensor dx = Tensor::empty(s, g.shape());
    s->check(vtlb_dropout_bwd_f32(s->ctx, g.data(), dx.data(), g.size(), mask.p, mask.seed, mask.step));
    return {dx};
  }
};

struct GroupNormGate : Gate {
  VarPtr input, gamma, beta;
  Tensor mean, rstd;
  int B, S, C, groups, act;
  std::vector<Tensor> backward(const Tensor& g) override {
    Session* s = g.session();
    Tensor dx, dgamma, dbeta;
    if (input->requires_grad) dx = Tensor::empty(s, input->value.shape());
    const bool params = gamma->requires_grad || beta->requires_grad;
    if (params) {  // one allocation, so that a data-parallel session reduces both with one collective
      const size_t off = ((size_t)C + 63) / 64 * 64;
      auto buf = std::make_shared<DeviceBuf>(s, 2 * off * sizeof(float));
      if (s->comm_on && off != (size_t)C) s->check(vtlb_memset0(s->ctx, buf->ptr, 2 * off * sizeof(float)));
      dgamma = Tensor::view(buf, 0, {1, C});
      dbeta = Tensor::view(buf, off, {1, C});
    }
    s->check(vtlb_groupnorm_bwd_f32(s->ctx, g.data(), input->value.data(), B, S, C, groups, gamma->value.data(),
                                    beta->value.data(), mean.data(), rstd.data(), act, dx.defined() ? dx.data() : nullptr,
                                    params ? dgamma.data() : nullptr, params ? dbeta.data() : nullptr));
    if (params && s->comm_on)
      s->check(vtlb_allreduce_sum_f32_async(s->ctx, dgamma.data(), dbeta.offset() + dbeta.size()));
    return {dx, gamma->requires_grad ? dgamma : Tensor(), beta->requires_grad ? dbeta : Tensor()};
  }
};

}  // namespace

// ---------------------------------------------------------------- embedding
EmbeddingLayer::EmbeddingLayer(Context* ctx, std::vector<int> in, int vocabulary_, int dim_, float scale_)
    : in_shape(std::move(in)), vocabulary(vocabulary_), dim(dim_), scale(scale_) {
  if (vocabulary <= 0 || dim <= 0) throw Error(VTLB_EINVAL, "EmbeddingLayer: vocabulary and dimension must be positive");
  if (vocabulary > (1 << 24) + 1) throw Error(VTLB_EINVAL, "EmbeddingLayer: tokens arrive as f32, which holds whole numbers to 2^24");
  Session* s = ctx->device_session;
  Tensor w = Tensor::empty(s, {vocabulary, dim});
  s->check(vtlb_init_normal_f32(s->ctx, w.data(), w.size(), 0.0, 1.0, s->next_init_seed()));
  weights = ctx->variable(w);
}
std::vector<int> EmbeddingLayer::output_shape() const {
  std::vector<int> out = in_shape;
  out.push_back(dim);
  return out;
}
VarPtr EmbeddingLayer::run(const VarPtr& input, const DropoutLayer::Mask& mask) {
  Context* ctx = input->context;
  Session* s = ctx->device_session;
  std::vector<int> shape = input->value.shape();
  const size_t n = count(shape);
  auto ids = std::make_shared<DeviceBuf>(s, n * sizeof(int32_t));
  s->check(vtlb_ids_from_f32(s->ctx, input->value.data(), n, ids->ptr));
  shape.push_back(dim);
  Tensor y = Tensor::empty(s, shape);
  s->check(vtlb_embedding_fwd_f32(s->ctx, weights->value.data(), vocabulary, dim, ids->ptr, n, scale, mask.p, mask.seed,
                                  mask.step, y.data(), 0));
  VarPtr out = ctx->variable(y);
  auto g = std::make_unique<EmbeddingGate>();
  g->weight = weights;
  g->ids = ids;
  g->n = n;
  g->scale = scale;
  g->mask = mask;
  ctx->register_node("Embedding", std::move(g), out, {input, weights});
  return out;
}
VarPtr EmbeddingLayer::forward(const VarPtr& input) { return run(input, DropoutLayer::Mask{}); }
VarPtr EmbeddingLayer::forward_with_dropout(const VarPtr& input, DropoutLayer& d) { return run(input, d.next_mask(input->context)); }

// ---------------------------------------------------------------- dropout
DropoutLayer::DropoutLayer(Context* ctx, std::vector<int> s, double p_) : shape(std::move(s)), p(p_) {
  if (!(p >= 0.0 && p <= 1.0)) throw Error(VTLB_EINVAL, "DropoutLayer: the probability must be in [0, 1]");
  // a key of its own per layer, and per rank: ranks hold different rows of a batch
  Session* ss = ctx->device_session;
  seed = ss->next_init_seed();
}
DropoutLayer::Mask DropoutLayer::next_mask(Context* ctx) {
  if (ctx->no_grad) return Mask{};  // inference: nothing is dropped, and no step is taken
  return Mask{p, seed + (uint64_t)ctx->device_session->rank * 0xD1B54A32D192ED03ull, step++};
}
VarPtr DropoutLayer::forward(const VarPtr& input) {
  Context* ctx = input->context;
  Session* s = ctx->device_session;
  const Mask mask = next_mask(ctx);
  if (mask.p == 0.0) return input;
  Tensor y = Tensor::empty(s, input->value.shape());
  s->check(vtlb_dropout_fwd_f32(s->ctx, input->value.data(), y.data(), y.size(), mask.p, mask.seed, mask.step));
  VarPtr out = ctx->variable(y);
  auto g = std::make_unique<DropoutGate>();
  g->mask = mask;
  ctx->register_node("Dropout", std::move(g), out, {input});
  return out;
}

// ---------------------------------------------------------------- group norm
GroupNormLayer::GroupNormLayer(Context* ctx, std::vector<int> in, int groups_, GroupNormConfig c)
    : in_shape(std::move(in)), groups(groups_), eps(c.eps), activation(c.activation) {
  if (in_shape.empty()) throw Error(VTLB_EINVAL, "GroupNormLayer: the input needs channels");
  channels = in_shape.back();
  if (groups <= 0 || channels % groups) throw Error(VTLB_EINVAL, "GroupNormLayer: the groups must divide the channels");
  if (!(eps >= 0.0)) throw Error(VTLB_EINVAL, "GroupNormLayer: eps must not be negative");
  if (activation < VTLB_ACT_NONE || activation > VTLB_ACT_SILU) throw Error(VTLB_EINVAL, "GroupNormLayer: unknown activation");
  Session* s = ctx->device_session;
  gamma = ctx->variable(Tensor::ones(s, {1, channels}));
  beta = ctx->variable(Tensor::zeros(s, {1, channels}));
}
VarPtr GroupNormLayer::forward(const VarPtr& input) {
  Context* ctx = input->context;
  Session* s = ctx->device_session;
  const auto& xs = input->value.shape();
  if (xs.size() < 2 || xs[0] <= 0 || xs.back() != channels)
    throw Error(VTLB_EINVAL, "GroupNormLayer.forward: input must be [batch, ..., channels]");
  const int B = xs[0], S = (int)(input->value.size() / B / channels);
  Tensor y = Tensor::empty(s, xs), mean = Tensor::empty(s, {B, groups}), rstd = Tensor::empty(s, {B, groups});
  s->check(vtlb_groupnorm_fwd_f32(s->ctx, input->value.data(), B, S, channels, groups, gamma->value.data(),
                                  beta->value.data(), eps, activation, y.data(), mean.data(), rstd.data()));
  VarPtr out = ctx->variable(y);
  auto g = std::make_unique<GroupNormGate>();
  g->input = input;
  g->gamma = gamma;
  g->beta = beta;
  g->mean = mean;
  g->rstd = rstd;
  g->B = B, g->S = S, g->C = channels, g->groups = groups, g->act = activation;
  ctx->register_node("GroupNorm", std::move(g), out, {input, gamma, beta});
  return out;
}

// ---------------------------------------------------------------- Sequential builders
void Sequential::embedding(int vocabulary, int dim, double scale) {
  for (const auto& l : layers)  // no gradient goes through tokens
    if (std::strcmp(l->kind(), "input")) throw Error(VTLB_EINVAL, "Sequential.embedding: takes tokens, so it follows the input");
  layers.push_back(std::make_unique<EmbeddingLayer>(&ctx_, cur_shape(), vocabulary, dim, (float)scale));
}
void Sequential::dropout(double p) { layers.push_back(std::make_unique<DropoutLayer>(&ctx_, cur_shape(), p)); }
void Sequential::groupnorm(int groups, GroupNormConfig c) {
  const auto sh = cur_shape();
  for (const auto& l : layers) {  // [C, H, W] of the image layers: their channels come first
    const char* k = l->kind();
    if (sh.size() == 3 && (!std::strcmp(k, "conv2d") || !std::strcmp(k, "maxpool2d") || !std::strcmp(k, "avgpool2d") ||
                           !std::strcmp(k, "global_avgpool2d")))
      throw Error(VTLB_EINVAL, "Sequential.groupnorm: takes [..., channels]; convolutions and pools leave [channels, H, W]");
  }
  layers.push_back(std::make_unique<GroupNormLayer>(&ctx_, sh, groups, c));
}

}  // namespace vtl
