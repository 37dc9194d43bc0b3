// INT8 linear layers on FP16 activations that are quantised token by token: the quantiser and the token-scaled layer behind it.
#include "device_utils.hpp"
#include "host_utils.hpp"
#include "network_ops.hpp"
#include "token_ops.hpp"
#include "trtamd_encoder_ops.h"

namespace trtamd
{
namespace
{

// The workspace of a dynamic layer: the quantised tokens, then their scales.
size_t quantized_bytes(int32_t T, int32_t K)
{
    return ((size_t) T * K + 255) / 256 * 256;
}

} // namespace
} // namespace trtamd

using namespace trtamd;

extern "C" size_t trtamd_int8_dynamic_linear_workspace_size(int32_t T, int32_t K, int32_t N)
{
    return T > 0 && K > 0 && N > 0 ? quantized_bytes(T, K) + (size_t) T * sizeof(float) : 0;
}

extern "C" int trtamd_int8_dynamic_linear(trtamd_stream_t stream, trtamd_int8_dynamic_linear_params const* p)
{
    if (p == nullptr)
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "int8_dynamic_linear: null pointer");
    }
    if (p->T > 0
        && (p->workspace == nullptr || !aligned16(p->workspace)
            || p->workspace_bytes < trtamd_int8_dynamic_linear_workspace_size(p->T, p->K, p->N)))
    {
        return set_error(TRTAMD_STATUS_BAD_PARAM, "int8_dynamic_linear: T=%d K=%d N=%d need a 16-byte aligned workspace of %zu bytes",
            p->T, p->K, p->N, trtamd_int8_dynamic_linear_workspace_size(p->T, p->K, p->N));
    }
    int8_t* const quantized = static_cast<int8_t*>(p->workspace);
    float* const scales = p->T > 0 ? reinterpret_cast<float*>(quantized + quantized_bytes(p->T, p->K)) : nullptr;
    trtamd_int8_token_linear_params const q = {quantized, p->w, scales, p->channel_scale, p->bias, p->out, p->T, p->K, p->N, p->epilogue};
    int st = int8_token_linear_check(q);
    st = st ? st : token_quantize_check("int8_dynamic_linear", p->T, p->K, p->a, p->a_stride, quantized, scales);
    if (st || p->T == 0)
    {
        return st;
    }
    st = token_quantize(stream, p->T, p->K, p->a, p->a_stride, quantized, scales);
    return st ? st : trtamd_int8_token_linear(stream, &q);
}
