// Device-side pieces that the kernels of the paged cache share: element types and row access.
#pragma once

#include "pqa_device.h"
#include "pqa_paged.h"

namespace pqa {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// The type of a handle: what the token rows and the pages hold.
template <int TYPE>
struct PagedType;
template <>
struct PagedType<PQA_PAGED_F32> {
    typedef float Io;
    typedef _Float16 Page;
};
template <>
struct PagedType<PQA_PAGED_F16> {
    typedef _Float16 Io;
    typedef _Float16 Page;
};
template <>
struct PagedType<PQA_PAGED_BF16> {
    typedef __bf16 Io;
    typedef __bf16 Page;
};

// fp32 to a page's type: fp16 with the reference's rounding (nearest, ties away from zero), as
// the contiguous cache's rows have it; bf16 to nearest, ties to even. Half a step of the type.
template <class Page>
__device__ __forceinline__ uint16_t to_page(float x) {
    if constexpr (__is_same(Page, _Float16)) return f32_to_f16_ref(x);
    else return __builtin_bit_cast(uint16_t, (__bf16)x);
}
template <class Page>
__device__ __forceinline__ float from_page(uint16_t x) {
    return (float)__builtin_bit_cast(Page, x);
}

// four elements of a row as fp32; `vec`: the row's start is aligned to four elements. ONCE: past
// the caches
template <class Io, bool ONCE = false>
__device__ __forceinline__ float4 load4(const Io* p, bool vec) {
    typedef Io v4 __attribute__((ext_vector_type(4)));
    if (vec) {
        const v4 x = ONCE ? __builtin_nontemporal_load((const v4*)p) : *(const v4*)p;
        return float4{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
    }
    return float4{(float)p[0], (float)p[1], (float)p[2], (float)p[3]};
}
template <class Io, bool ONCE = false>
__device__ __forceinline__ void store4(Io* p, float4 x, bool vec) {
    typedef Io v4 __attribute__((ext_vector_type(4)));
    const v4 y = {(Io)x.x, (Io)x.y, (Io)x.z, (Io)x.w};
    if (vec) {
        if constexpr (ONCE) __builtin_nontemporal_store(y, (v4*)p);
        else *(v4*)p = y;
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) p[e] = y[e];
}

// floor(log2(x)) of x >= 0, within [-24, 24]; 24 for infinities and NaN, -24 for zero
__device__ __forceinline__ int bound_exponent(float x) {
    return min(max((int)((__float_as_uint(x) >> 23) & 0xFFu) - 127, -24), 24);
}
__device__ __forceinline__ float power2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// 16 bytes per lane from the lane's own global address straight into LDS (lane l's bytes land
// at lds + 16 l); the contract of lds_dma_b128.
__device__ __forceinline__ void lds_dma_b128_at(const void* p, unsigned lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(lds) : "memory", "m0");
}

// Called by the whole workgroup after its part's stores (agent scope, relaxed: past the L2s, which are
// not coherent between dies); true in the workgroup that finishes last, which then sees all
// parts. Its counter is zero again for the next call.
__device__ __forceinline__ bool last_of(unsigned* counter, int parts, int* flag) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores have reached memory
    __syncthreads();
    if (threadIdx.x == 0) {
        const unsigned n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *flag = n == (unsigned)parts - 1;
        if (*flag) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    asm volatile("" ::: "memory");  // the loads of the parts stay behind the counter
    return *flag != 0;
}

// a table that the kernel only reads, through the scalar cache
typedef const __attribute__((address_space(4))) int* ScalarInts;
__device__ __forceinline__ int scalar_int(const int* p, int i) {
    return ((ScalarInts)(unsigned long long)p)[__builtin_amdgcn_readfirstlane(i)];
}

}  // namespace pqa
