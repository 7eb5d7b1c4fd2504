// Shared between the training operators (train_embed.hip, train_clip.hip, train_head.hip, swiglu.hip): vectors of the three storage types as fp32 values.
#pragma once
#include <type_traits>
#include "common.h"
#include "../../include/videoitg_hip.h"

namespace vitg {

// V consecutive elements of type T <-> fp32 values; p aligned to the vector, or to 16 bytes where the vector is longer (eight fp32 values: two 16-byte accesses) -
// what the entry points check
template <typename T, int V> struct Pack {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T) * V < 16 ? sizeof(T) * V : 16)));
};
static_assert(alignof(Pack<float, 8>::type) == 16 && alignof(Pack<bf16_t, 8>::type) == 16 && alignof(Pack<f16_t, 4>::type) == 8 && sizeof(Pack<float, 8>::type) == 32,
              "no access asks for more than the checked alignment");
template <typename T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
    const typename Pack<T, V>::type x = *(const typename Pack<T, V>::type*)p;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)x[i];
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
    typename Pack<T, V>::type x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (T)v[i];
    *(typename Pack<T, V>::type*)p = x;
}
// Streams that do not fit the 256 MB last-level cache go around it (non-temporal): what they displace - and the write-back of what they leave dirty - costs the
// next kernel more than it saves.  A tensor of up to half of it keeps the ordinary form: its next reader finds it there.
constexpr long STREAM_BYTES = 128l << 20;
// (template arguments, not run-time flags: two stores that differ only in the hint are merged by the compiler, and the hint is lost)
template <typename T, int V, bool AROUND> __device__ __forceinline__ void store_stream(T* p, const float (&v)[V]) {
    typename Pack<T, V>::type x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (T)v[i];
    if constexpr (AROUND) __builtin_nontemporal_store(x, (typename Pack<T, V>::type*)p);
    else *(typename Pack<T, V>::type*)p = x;
}
template <typename T, int V, bool AROUND> __device__ __forceinline__ void load_stream(const T* p, float (&v)[V]) {
    typename Pack<T, V>::type x;
    if constexpr (AROUND) x = __builtin_nontemporal_load((const typename Pack<T, V>::type*)p);
    else x = *(const typename Pack<T, V>::type*)p;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)x[i];
}

inline bool dtype_ok(int dt) { return dt == DT_BF16 || dt == DT_F16 || dt == DT_F32; }
inline int dtype_size(int dt) { return dt == DT_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }
inline int launched() { return hipGetLastError() == hipSuccess ? 0 : VITG_ERR_LAUNCH; }

// f(std::true_type{}) / f(std::false_type{})
template <typename F> inline auto with_flag(bool on, F f) { return on ? f(std::true_type{}) : f(std::false_type{}); }
// f(T{}) for the storage type of a dtype code that dtype_ok() has accepted
template <typename F> inline auto with_dtype(int dt, F f) { return dt == DT_BF16 ? f(bf16_t{}) : dt == DT_F16 ? f(f16_t{}) : f(float{}); }

}  // namespace vitg
