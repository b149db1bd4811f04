// The 16-bit products' kernels of one operand type: compiled with FEATHER_LINEAR_BF16 set to 0 (fp16) or 1 (bf16).
#include "linear_few.h"
#include "linear_launch.h"
#include "linear_tile.h"

namespace feather {
namespace {

constexpr bool kBf16 = FEATHER_LINEAR_BF16 != 0;

template <typename T, bool kAAcross, bool kBAcross, Form kForm>
void tile(const LinearParams& p, const LinearPlan& plan, hipStream_t stream) {
    linear_tile_kernel<T, kAAcross, kBAcross, kForm, kBf16>
        <<<static_cast<uint32_t>(plan.tiles * plan.splits), T::kThreads, 0, stream>>>(p);
}

template <bool kAAcross, bool kBAcross, Form kForm>
void tiles(const LinearParams& p, const LinearPlan& plan, hipStream_t stream) {
    if (plan.kernel == kTile256) tile<LinearTile<256, 256>, kAAcross, kBAcross, kForm>(p, plan, stream);
    else if (plan.kernel == kTile256x128) tile<LinearTile<256, 128>, kAAcross, kBAcross, kForm>(p, plan, stream);
    else tile<LinearTile<128, 128>, kAAcross, kBAcross, kForm>(p, plan, stream);
}

template <typename T, Form kForm>
void few(const LinearParams& p, const LinearPlan& plan, hipStream_t stream) {
    few_rows_kernel<T, 0, false, kForm, kBf16>
        <<<dim3(static_cast<uint32_t>(plan.tiles), plan.splits), T::kThreads, 0, stream>>>(p);
}

template <Form kForm>
void gated(const LinearParams& p, const LinearPlan& plan, hipStream_t stream) {
    if (plan.kernel == kFew16_2_8_1) few<FewRows<1, 2, 8, 1>, kForm>(p, plan, stream);
    else if (plan.kernel == kFew16_2_4_2) few<FewRows<1, 2, 4, 2>, kForm>(p, plan, stream);
    else if (plan.kernel == kFew32_4_4_2) few<FewRows<2, 4, 4, 2>, kForm>(p, plan, stream);
    else if (plan.kernel == kFew32_2_4_2) few<FewRows<2, 2, 4, 2>, kForm>(p, plan, stream);
    else if (plan.kernel == kFew64_2_4_2) few<FewRows<4, 2, 4, 2>, kForm>(p, plan, stream);
    else tiles<false, false, kForm>(p, plan, stream);
}

}  // namespace

#if FEATHER_LINEAR_BF16
#define FEATHER_LAUNCH linear_launch_bf16
#else
#define FEATHER_LAUNCH linear_launch_fp16
#endif

void FEATHER_LAUNCH(const LinearParams& p, const LinearPlan& plan, Operands operands, hipStream_t stream) {
    if (operands == Operands::kGated) gated<Form::kGated>(p, plan, stream);
    else if (operands == Operands::kGatedKeep) gated<Form::kGatedKeep>(p, plan, stream);
    else if (operands == Operands::kAlong) tiles<false, false, Form::kPlain>(p, plan, stream);
    else if (operands == Operands::kBAcross) tiles<false, true, Form::kPlain>(p, plan, stream);
    else tiles<true, true, Form::kPlain>(p, plan, stream);
}

}  // namespace feather
