// The join of products whose K is split over workgroups.
#pragma once

#include "scaled_mm_kernels.h"

namespace feather {

// A tile whose K is split over p.splits workgroups: parts of it (kSlots a tile, each one wave's fp32 sums) meet in the
// workspace. A wave writes its sums through to the memory that all XCDs share, counts itself in, and the last of the part's
// waves to come reads all of them back, adds them in order of the K ranges (so the result does not depend on who was last),
// leaves the counter at zero and returns true: it stores the outputs. Nobody waits for another workgroup.
template <int kSlots, typename P, int RM, int RN>
__device__ __forceinline__ bool join_splits(const P& p, f32x4 (&acc)[RM][RN], int tile, int split, int slot,
                                            int lane) {
    constexpr uint32_t kPartBytes = RM * RN * kWave * 16;
    const rsrc_t parts = make_rsrc(p.split_part, 0x7fffffffu);
    const auto place = [&](int s) {
        return (static_cast<uint32_t>(tile * p.splits + s) * kSlots + slot) * kPartBytes + lane * 16u;
    };
    uint32_t* const counter = p.split_ctr + tile * kSlots + slot;
#pragma unroll
    for (int f = 0; f < RM * RN; ++f)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[f / RN][f % RN]), parts,
                                               place(split) + f * kWave * 16u, 0, kDeviceScope);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // written for every XCD before the count says so
    uint32_t before = 0;
    if (lane == 0) before = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    before = __builtin_amdgcn_readfirstlane(before);
    asm volatile("" ::: "memory");   // the reads below come after it
    if (before + 1 != static_cast<uint32_t>(p.splits)) return false;
    constexpr int kFragments = RM * RN;
    constexpr int kBatch = kFragments % 16 == 0 ? 16 : kFragments;
    const auto load = [&](f32x4 (&part)[kBatch], int s, int f0) {
#pragma unroll
        for (int f = 0; f < kBatch; ++f) {
            const uint32_t at = place(s) + (f0 + f) * kWave * 16u;
            part[f] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(parts, at, 0, kDeviceScope));
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // As many loads in flight as there are registers for. (The block-scaled products, 71 split shapes of 1 to 4096 rows, take as long as
    // with a loop over the parts alone: 1.000 of its time in the mean, 0.986 to 1.015.) (Left to itself the compiler waits for each: 1000 x 27648 x 5120 in 256 x
    // 256 tiles and three K ranges took 266 us, with 16 together 257.) Where a SIMD has one wave there is room for two batches: one
    // is loaded while the other is added.
    const auto add = [&](const f32x4 (&part)[kBatch], int s, int f0) {
#pragma unroll
        for (int f = 0; f < kBatch; ++f) {
            f32x4& sum = acc[(f0 + f) / RN][(f0 + f) % RN];
            sum = s == 0 ? part[f] : sum + part[f];
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (kFragments == 4 * kBatch) {
        f32x4 even[kBatch], odd[kBatch];
        load(even, 0, 0);
        for (int s = 0; s < p.splits; ++s) {
            load(odd, s, kBatch);
            add(even, s, 0);
            load(even, s, 2 * kBatch);
            add(odd, s, kBatch);
            load(odd, s, 3 * kBatch);
            add(even, s, 2 * kBatch);
            load(even, s + 1 < p.splits ? s + 1 : s, 0);   // (the last one for nothing)
            add(odd, s, 3 * kBatch);
        }
    } else {
        for (int s = 0; s < p.splits; ++s) {
#pragma unroll
            for (int f0 = 0; f0 < kFragments; f0 += kBatch) {
                f32x4 part[kBatch];
                load(part, s, f0);
                add(part, s, f0);
            }
        }
    }
    if (lane == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

}  // namespace feather
