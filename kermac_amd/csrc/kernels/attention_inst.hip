// Instantiations of the attention kernels for one element type (KMC_ATT_TYPE: 0 fp32, 1 fp16, 2 bf16).
#include "attention.hpp"
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

template <int DP>
hipError_t forward(const kmc::AttentionArgs &args, bool aligned, hipStream_t stream)
{
    return launch_in_parts(aligned ? kmc::attention_forward<Element, DP, true> : kmc::attention_forward<Element, DP, false>, args.job[0].grid + args.job[1].grid,
                           kmc::ATT_MAX_BLOCKS, dim3(256), stream, args);
}

}  // namespace

#define KMC_ATT_NAME_2(name, type) name##_##type
#define KMC_ATT_NAME_1(name, type) KMC_ATT_NAME_2(name, type)
#define KMC_ATT_NAME(name) KMC_ATT_NAME_1(name, KMC_ATT_TYPE)

hipError_t KMC_ATT_NAME(launch_attention_forward)(const kmc::AttentionArgs &args, int width, bool aligned, hipStream_t stream)
{
    if (args.job[0].grid + args.job[1].grid > 0) {
        const hipError_t status = width <= 64 ? forward<64>(args, aligned, stream) : width <= 96 ? forward<96>(args, aligned, stream) : width <= 128 ? forward<128>(args, aligned, stream)
                                                                                                  : forward<256>(args, aligned, stream);
        if (status != hipSuccess) return status;
    }
    if (args.slots == 0) return hipSuccess;
    const kmc::i64 blocks = (args.rows_total + 3) / 4;
    return launch(kmc::attention_join<Element>, dim3(static_cast<unsigned>(blocks < kmc::ATT_MAX_BLOCKS ? blocks : kmc::ATT_MAX_BLOCKS)), dim3(256), stream, args);
}

}  // namespace kmc_host
