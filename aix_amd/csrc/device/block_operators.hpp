// block_operators.hpp -- operators of transformer blocks that a device may offer beside aix::Device's own: attention with
// windows and leading keys, rotary positions, matrix products with an epilogue, and their gradients.  The reference composes
// them from Device's operators (aixNeuralNetwork.hpp:182-208); a caller asks a device for them with
// dynamic_cast<aix::hip::BlockOperators*>(device).  Meanings, shapes and limits: include/aixhip_kernels.h, the entry points of
// the same names.
#pragma once

#include "aix_compat.hpp"

namespace aix::hip {

struct AttentionSpec {
    float scale{1.0f};                              // factor of the scores, positive
    bool causal{true};
    size_t window{0}, sinks{0};                     // window 0: none; sinks: leading keys that a window does not hide
    const DeviceTensorParams* lengths{nullptr};     // int32 [batch]: keys in use; null: all
    const DeviceTensorParams* starts{nullptr};      // int32 [batch]: position of the first query; null: the queries are the last ones
};

enum class RotaryScaling { kPlain, kLinear, kBase, kParts };
struct RotarySpec {
    size_t dims{0};                                 // leading elements of every head that are turned
    bool interleaved{false}, inverse{false};
    RotaryScaling scaling{RotaryScaling::kPlain};
    double base{10000.0}, factor{1.0}, originalLength{1.0}, lowTurns{1.0}, highTurns{32.0};
    float magnitude{1.0f};
};

enum class Activation { kNone, kReLU, kGELU, kSiLU };
struct Epilogue {
    const DeviceTensorParams* bias{nullptr};        // [N] or [1, N]
    const DeviceTensorParams* residual{nullptr};    // [M, N]
    const DeviceTensorParams* pre{nullptr};         // [M, N], receives product + bias
    Activation activation{Activation::kNone};
};

class BlockOperators {
public:
    virtual ~BlockOperators() = default;
    virtual void attention(const DeviceTensorParams& q, const DeviceTensorParams& k, const DeviceTensorParams& v, const AttentionSpec& spec,
                           const DeviceTensorParams& result, const DeviceTensorParams* lse) = 0;
    virtual void attentionBackward(const DeviceTensorParams& grad, const DeviceTensorParams& q, const DeviceTensorParams& k, const DeviceTensorParams& v,
                                   const DeviceTensorParams& out, const DeviceTensorParams& lse, const AttentionSpec& spec,
                                   const DeviceTensorParams& dq, const DeviceTensorParams& dk, const DeviceTensorParams& dv) = 0;
    // k and kResult may be null
    virtual void rotary(const DeviceTensorParams& q, const DeviceTensorParams* k, const DeviceTensorParams& positions, const RotarySpec& spec,
                        const DeviceTensorParams& qResult, const DeviceTensorParams* kResult) = 0;
    virtual void matmulEpilogue(const DeviceTensorParams& a, const DeviceTensorParams& b, const Epilogue& epilogue, const DeviceTensorParams& result) = 0;
    // pre, dz, da, db, dbias may be null as for aixk_matmul_epilogue_backward
    virtual void matmulEpilogueBackward(const DeviceTensorParams& grad, const DeviceTensorParams& a, const DeviceTensorParams& b, const DeviceTensorParams* pre,
                                        Activation activation, const DeviceTensorParams* dz, const DeviceTensorParams* da, const DeviceTensorParams* db,
                                        const DeviceTensorParams* dbias) = 0;
};

} // namespace aix::hip
