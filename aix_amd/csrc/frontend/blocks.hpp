// blocks.hpp -- a device's transformer-block operators (device/block_operators.hpp) as differentiable functions of
// aixfe::Tensor: attention, rotary positions and a linear layer with activation and residual.  A device without them
// (the CPU oracle) is refused with std::invalid_argument; programs for any device compose them from Tensor's operators.
#pragma once

#include "autograd.hpp"
#include "../device/block_operators.hpp"

namespace aixfe {

using aix::hip::Activation;
using aix::hip::BlockOperators;

inline BlockOperators& blockOperators(Device* dev)
{
    auto* ops = dynamic_cast<BlockOperators*>(dev);
    if (!ops) throw std::invalid_argument("this device has no transformer-block operators");
    return *ops;
}

inline void requireRank(const Tensor& t, size_t rank, const char* what)
{
    if (t.shape().size() != rank) throw std::invalid_argument(what);
}

// [batch, heads, sequence, head dim] over memory [batch, sequence, heads, head dim]: what projections leave and take
inline Value headsOf(Device* dev, DataType dt, const Shape& s) { return Value(dev, dt, Shape{s[0], s[2], s[1], s[3]}).transpose(1, 2); }

// Which keys a query sees and how its scores are scaled (aix::hip::AttentionSpec with values in place of descriptors).
struct AttentionMask {
    float scale{1.0f};
    bool causal{true};
    size_t window{0}, sinks{0};
    Value lengths, starts;                 // int32 [batch], or undefined
    aix::hip::AttentionSpec spec() const
    {
        return {scale, causal, window, sinks, lengths.defined() ? &lengths.params() : nullptr, starts.defined() ? &starts.params() : nullptr};
    }
};

// q [batch, heads, queries, d], k and v [batch, key heads, keys, d] -> like q
inline Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const AttentionMask& mask)
{
    for (const Tensor* t : {&q, &k, &v}) requireRank(*t, 4, "attention: queries, keys and values must be [batch, heads, sequence, head dim]");
    Device* dev = q.device();
    const Shape& s = q.shape();
    const Value out = headsOf(dev, q.dtype(), s), lse(dev, DataType::kFloat32, Shape{s[0], s[1], s[2]});
    blockOperators(dev).attention(q.value().params(), k.value().params(), v.value().params(), mask.spec(), out.params(), &lse.params());
    return Tensor::fromOperator(out, {q, k, v}, [out, lse, mask](Node* n, const Value& seed) {
        if (n->inputs.size() < 3) return;
        Device* d = seed.device();
        const Value &vq = n->inputs[0]->value, &vk = n->inputs[1]->value, &vv = n->inputs[2]->value;
        const Value dq = headsOf(d, seed.dtype(), vq.shape()), dk = headsOf(d, seed.dtype(), vk.shape()), dv = headsOf(d, seed.dtype(), vv.shape());
        blockOperators(d).attentionBackward(seed.params(), vq.params(), vk.params(), vv.params(), out.params(), lse.params(), mask.spec(), dq.params(), dk.params(), dv.params());
        if (Tensor::wants(n->inputs[0])) n->inputs[0]->backward(dq);
        if (Tensor::wants(n->inputs[1])) n->inputs[1]->backward(dk);
        if (Tensor::wants(n->inputs[2])) n->inputs[2]->backward(dv);
    }, 7);
}

// queries and keys turned by their positions (int32 [batch, sequence]), in one call
inline std::pair<Tensor, Tensor> rotary(const Tensor& q, const Tensor& k, const Value& positions, const aix::hip::RotarySpec& spec)
{
    for (const Tensor* t : {&q, &k}) requireRank(*t, 4, "rotary: queries and keys must be [batch, heads, sequence, head dim]");
    Device* dev = q.device();
    const Value tq = headsOf(dev, q.dtype(), q.shape()), tk = headsOf(dev, k.dtype(), k.shape());
    blockOperators(dev).rotary(q.value().params(), &k.value().params(), positions.params(), spec, tq.params(), &tk.params());
    auto back = [positions, spec](Node* n, const Value& seed) {
        if (n->inputs.empty()) return;
        aix::hip::RotarySpec turn = spec;
        turn.inverse = !spec.inverse;
        const Value g = headsOf(seed.device(), seed.dtype(), seed.shape());
        blockOperators(seed.device()).rotary(seed.params(), nullptr, positions.params(), turn, g.params(), nullptr);
        n->inputs[0]->backward(g);
    };
    return {Tensor::fromOperator(tq, {q}, back, 0), Tensor::fromOperator(tk, {k}, back, 0)};
}

// act(x . w + b) [+ residual]: x [rows, in], w [in, out], b [1, out]
inline Tensor linear(const Tensor& x, const Tensor& w, const Tensor& b, Activation act = Activation::kNone, const Tensor* residual = nullptr)
{
    for (const Tensor* t : {&x, &w}) requireRank(*t, 2, "linear: rows and weights must be 2-D");
    Device* dev = x.device();
    const Shape s{x.shape()[0], w.shape()[1]};
    const Value out(dev, x.dtype(), s), pre = act != Activation::kNone ? Value(dev, x.dtype(), s) : Value();
    blockOperators(dev).matmulEpilogue(x.value().params(), w.value().params(),
                                       {&b.value().params(), residual ? &residual->value().params() : nullptr, pre.defined() ? &pre.params() : nullptr, act}, out.params());
    std::vector<Tensor> inputs{x, w, b};
    if (residual) inputs.push_back(*residual);
    return Tensor::fromOperator(out, inputs, [pre, act](Node* n, const Value& seed) {
        if (n->inputs.size() < 3) return;
        Device* d = seed.device();
        const Value &vx = n->inputs[0]->value, &vw = n->inputs[1]->value;
        const bool wx = Tensor::wants(n->inputs[0]), ww = Tensor::wants(n->inputs[1]), wb = Tensor::wants(n->inputs[2]);
        Value dz, dx, dw, db;
        if (act != Activation::kNone) dz = Value(d, seed.dtype(), seed.shape());
        if (wx) dx = Value(d, seed.dtype(), vx.shape());
        if (ww) dw = Value(d, seed.dtype(), vw.shape());
        if (wb) db = Value(d, seed.dtype(), n->inputs[2]->value.shape());
        auto maybe = [](const Value& v) { return v.defined() ? &v.params() : nullptr; };
        blockOperators(d).matmulEpilogueBackward(seed.params(), vx.params(), vw.params(), maybe(pre), act, maybe(dz), maybe(dx), maybe(dw), maybe(db));
        if (wx) n->inputs[0]->backward(dx);
        if (ww) n->inputs[1]->backward(dw);
        if (wb) n->inputs[2]->backward(db);
        if (n->inputs.size() > 3 && Tensor::wants(n->inputs[3])) n->inputs[3]->backward(seed);
    }, 3);
}

} // namespace aixfe
