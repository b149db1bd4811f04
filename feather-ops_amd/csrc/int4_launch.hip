// The 4-bit products' kernels of one activation type: compiled with FEATHER_LINEAR_BF16 set to 0 (fp16) or 1 (bf16).
#include "int4_tile.h"
#include "linear_few.h"
#include "linear_launch.h"

namespace feather {
namespace {

constexpr bool kBf16 = FEATHER_LINEAR_BF16 != 0;

template <typename T, int kGroups, bool kZeros, Form kForm>
void few(const Int4Params& p, const LinearPlan& plan, hipStream_t stream) {
    few_rows_kernel<T, kGroups, kZeros, kForm, kBf16>
        <<<dim3(static_cast<uint32_t>(plan.tiles), plan.splits), T::kThreads, 0, stream>>>(p);
}

template <int kGroups, bool kZeros>
void plain(const Int4Params& p, const LinearPlan& plan, hipStream_t stream) {
    constexpr Form kForm = Form::kPlain;
    if (plan.kernel == kFew16_1_16_1) few<FewRows<1, 1, 16, 1>, kGroups, kZeros, kForm>(p, plan, stream);
    else if (plan.kernel == kFew16_1_8_2) few<FewRows<1, 1, 8, 2>, kGroups, kZeros, kForm>(p, plan, stream);
    else if (plan.kernel == kFew16_2_8_1) few<FewRows<1, 2, 8, 1>, kGroups, kZeros, kForm>(p, plan, stream);
    else if (plan.kernel == kFew32_1_4_4) few<FewRows<2, 1, 4, 4>, kGroups, kZeros, kForm>(p, plan, stream);
    else few<FewRows<4, 2, 4, 2>, kGroups, kZeros, kForm>(p, plan, stream);
}

template <int kGroups, bool kZeros>
void gated(const Int4Params& p, const LinearPlan& plan, hipStream_t stream) {
    constexpr Form kForm = Form::kGated;
    if constexpr (!kZeros || kGroups == 1 || (kGroups == 2 && !kBf16)) {   // others have no plan of 16 waves
        if (plan.kernel == kFew16_2_16_1) return few<FewRows<1, 2, 16, 1>, kGroups, kZeros, kForm>(p, plan, stream);
        if (plan.kernel == kFew32_2_4_4) return few<FewRows<2, 2, 4, 4>, kGroups, kZeros, kForm>(p, plan, stream);
    }
    if (plan.kernel == kFew16_2_4_2) few<FewRows<1, 2, 4, 2>, kGroups, kZeros, kForm>(p, plan, stream);
    else if (plan.kernel == kFew16_2_8_1) few<FewRows<1, 2, 8, 1>, kGroups, kZeros, kForm>(p, plan, stream);
    else if (plan.kernel == kFew32_2_4_2) few<FewRows<2, 2, 4, 2>, kGroups, kZeros, kForm>(p, plan, stream);
    else few<FewRows<4, 2, 4, 2>, kGroups, kZeros, kForm>(p, plan, stream);
}

template <Form kForm>
void tile(const Int4Params& p, const LinearPlan& plan, hipStream_t stream) {
    const dim3 groups(static_cast<uint32_t>(plan.tiles * plan.splits));
    if (plan.kernel == kInt4Tile256) int4_tile_kernel<Int4Tile<256>, kForm, kBf16><<<groups, Int4Tile<256>::kThreads, 0, stream>>>(p);
    else int4_tile_kernel<Int4Tile<128>, kForm, kBf16><<<groups, Int4Tile<128>::kThreads, 0, stream>>>(p);
}

template <int kGroups>
void by_group(const Int4Params& p, const LinearPlan& plan, bool gate, hipStream_t stream) {
    if (p.zero) (gate ? gated<kGroups, true> : plain<kGroups, true>)(p, plan, stream);
    else (gate ? gated<kGroups, false> : plain<kGroups, false>)(p, plan, stream);
}

}  // namespace

#if FEATHER_LINEAR_BF16
#define FEATHER_LAUNCH int4_launch_bf16
#else
#define FEATHER_LAUNCH int4_launch_fp16
#endif

void FEATHER_LAUNCH(const Int4Params& p, const LinearPlan& plan, bool gated, hipStream_t stream) {
    if (plan.kernel <= kInt4Tile128) (gated ? tile<Form::kGated> : tile<Form::kPlain>)(p, plan, stream);
    else if (p.group == 32) by_group<4>(p, plan, gated, stream);
    else if (p.group == 64) by_group<2>(p, plan, gated, stream);
    else by_group<1>(p, plan, gated, stream);
}

}  // namespace feather
