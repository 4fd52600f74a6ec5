// Instantiations of attention's gradient for one element type (KMC_ATT_TYPE: 0 fp32, 1 fp16, 2 bf16).
#include "attention_grad.hpp"
#include "launch.hpp"

namespace kmc_host {

namespace {

#if KMC_ATT_TYPE == 0
typedef float Element;
#elif KMC_ATT_TYPE == 1
typedef _Float16 Element;
#else
typedef __bf16 Element;
#endif

template <int DP, bool ALIGNED>
hipError_t gradient(const kmc::AttentionGradArgs &args, hipStream_t stream)
{
    // the queries' kernel writes delta, which the keys' kernel reads
    const hipError_t status = launch_in_parts(kmc::attention_grad_queries<Element, DP, ALIGNED>, args.q_grid, kmc::ATT_MAX_BLOCKS, dim3(256), stream, args);
    if (status != hipSuccess || args.k_grid == 0) return status;
    if constexpr (DP * sizeof(Element) > 512) {
        const hipError_t first = launch_in_parts(kmc::attention_grad_keys<Element, DP, ALIGNED, kmc::ATT_GRAD_KEYS>, args.k_grid, kmc::ATT_MAX_BLOCKS, dim3(256), stream, args);
        if (first != hipSuccess) return first;
        return launch_in_parts(kmc::attention_grad_keys<Element, DP, ALIGNED, kmc::ATT_GRAD_VALUES>, args.k_grid, kmc::ATT_MAX_BLOCKS, dim3(256), stream, args);
    } else {
        return launch_in_parts(kmc::attention_grad_keys<Element, DP, ALIGNED, kmc::ATT_BOTH>, args.k_grid, kmc::ATT_MAX_BLOCKS, dim3(256), stream, args);
    }
}

template <int DP>
hipError_t gradient(const kmc::AttentionGradArgs &args, bool aligned, hipStream_t stream)
{
    return aligned ? gradient<DP, true>(args, stream) : gradient<DP, false>(args, stream);
}

}  // namespace

#define KMC_ATT_NAME_2(name, type) name##_##type
#define KMC_ATT_NAME_1(name, type) KMC_ATT_NAME_2(name, type)
#define KMC_ATT_NAME(name) KMC_ATT_NAME_1(name, KMC_ATT_TYPE)

hipError_t KMC_ATT_NAME(launch_attention_gradient)(const kmc::AttentionGradArgs &args, int width, bool aligned, hipStream_t stream)
{
    hipError_t status = width <= 64    ? gradient<64>(args, aligned, stream)
                        : width <= 96  ? gradient<96>(args, aligned, stream)
                        : width <= 128 ? gradient<128>(args, aligned, stream)
                                       : gradient<256>(args, aligned, stream);
    if (status != hipSuccess || (args.q_splits == 1 && args.k_splits == 1)) return status;
    const kmc::i64 q_rows = static_cast<kmc::i64>(args.l) * args.m * args.g * args.r;
    const kmc::i64 k_rows = args.k_splits > 1 ? static_cast<kmc::i64>(args.key_entries) * args.keys.n * args.g : 0;
    const kmc::AttentionSum parts[3] = {
        {args.partial_q, args.grad_q, args.q_splits > 1 ? q_rows : 0, args.q_splits, args.k, args.partial_k_width, args.scale},
        {args.partial_k, args.grad_k, k_rows, args.k_splits, args.k, args.partial_k_width, args.scale},
        {args.partial_v, args.grad_v, k_rows, args.k_splits, args.o, args.partial_o_width, kmc::ATT_GRAD_LOWER<Element>}};
    kmc::AttentionSumArgs sums = {};
    for (int i = 0; i < 3; ++i) {
        sums.part[i] = parts[i];
        sums.first[i + 1] = sums.first[i] + parts[i].rows * parts[i].width;
    }
    const kmc::i64 blocks = (sums.first[3] + 255) / 256;
    if (blocks > 0) status = launch(kmc::attention_sum<Element>, dim3(static_cast<unsigned>(blocks < 16384 ? blocks : 16384)), dim3(256), stream, sums);
    return status;
}

}  // namespace kmc_host
