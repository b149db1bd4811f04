// The 4-bit products' kernels of one activation type: compiled with FEATHER_LINEAR_BF16 set to 0 (fp16) or 1 (bf16).
#include "linear_launch.h"
#include "linear_stream.h"

namespace feather {
namespace {

constexpr bool kBf16 = FEATHER_LINEAR_BF16 != 0;

template <int RM, int kGroups, bool kZeros, Form kForm>
void few(const Int4Params& p, const LinearPlan& plan, hipStream_t stream) {
    using T = LinearStream<RM, 2, 8, 2>;
    linear_stream_kernel<T, kGroups, kZeros, kForm, kBf16>
        <<<dim3(static_cast<uint32_t>(plan.tiles), plan.splits), T::kThreads, 0, stream>>>(p);
}

template <int kGroups, bool kZeros, Form kForm>
void by_rows(const Int4Params& p, const LinearPlan& plan, hipStream_t stream) {
    if (plan.kernel == kFewRows16) few<1, kGroups, kZeros, kForm>(p, plan, stream);
    else if (plan.kernel == kFewRows32) few<2, kGroups, kZeros, kForm>(p, plan, stream);
    else few<4, kGroups, kZeros, kForm>(p, plan, stream);
}

template <int kGroups>
void by_group(const Int4Params& p, const LinearPlan& plan, bool gated, hipStream_t stream) {
    if (p.zero) {
        if (gated) by_rows<kGroups, true, Form::kGated>(p, plan, stream);
        else by_rows<kGroups, true, Form::kPlain>(p, plan, stream);
    } else {
        if (gated) by_rows<kGroups, false, Form::kGated>(p, plan, stream);
        else by_rows<kGroups, false, Form::kPlain>(p, plan, stream);
    }
}

}  // namespace

#if FEATHER_LINEAR_BF16
#define FEATHER_LAUNCH int4_launch_bf16
#else
#define FEATHER_LAUNCH int4_launch_fp16
#endif

void FEATHER_LAUNCH(const Int4Params& p, const LinearPlan& plan, bool gated, hipStream_t stream) {
    if (p.group == 32) by_group<4>(p, plan, gated, stream);
    else if (p.group == 64) by_group<2>(p, plan, gated, stream);
    else by_group<1>(p, plan, gated, stream);
}

}  // namespace feather
