// Entry points called with their arguments in an array of 64-bit words.
#include <limits.h>

#include <type_traits>
#include <utility>

#include "q4_host.h"

namespace alv {
namespace {

// Word i as an argument of type A: pointers and integers as they are (an int's word
// within 32 bits), floats from a double.
template <class A>
A argument(uint64_t w) {
    if constexpr (std::is_pointer_v<A>) {
        return reinterpret_cast<A>(static_cast<uintptr_t>(w));
    } else if constexpr (std::is_floating_point_v<A>) {
        return static_cast<A>(__builtin_bit_cast(double, w));
    } else {
        return static_cast<A>(w);
    }
}

template <class A>
bool fits(uint64_t w) {
    if constexpr (std::is_same_v<A, int>) return static_cast<int64_t>(w) >= INT_MIN && static_cast<int64_t>(w) <= INT_MAX;
    return true;
}

template <class... A, size_t... I>
int call_with(int (*f)(A...), const uint64_t* w, std::index_sequence<I...>) {
    int bad = -1;
    ((fits<A>(w[I]) || bad >= 0 ? void() : void(bad = (int)I)), ...);
    if (bad >= 0) return fail(ALV_ERR_RANGE, "argument %d: %lld is past 32 bits", bad, (long long)w[bad]);
    return f(argument<A>(w[I])...);
}

template <class... A>
int call(int (*f)(A...), const uint64_t* w, int n) {
    if (n != (int)sizeof...(A)) return fail(ALV_ERR_ARG, "%d arguments, %d needed", n, (int)sizeof...(A));
    return call_with(f, w, std::index_sequence_for<A...>());
}

}  // namespace
}  // namespace alv

extern "C" int alv_call(int entry, const uint64_t* words, int n) {
    using namespace alv;
    if (!words) return fail(ALV_ERR_ARG, "null pointer");
    switch (entry) {
        case ALV_CALL_QKV_POST_PAGED: return call(alv_qkv_post_paged, words, n);
        case ALV_CALL_QKV_POST_PAGED8: return call(alv_qkv_post_paged8, words, n);
        case ALV_CALL_ATTENTION_PAGED: return call(alv_attention_paged, words, n);
        case ALV_CALL_ATTENTION_PAGED8: return call(alv_attention_paged8, words, n);
        case ALV_CALL_ATTENTION_SHARED: return call(alv_attention_shared, words, n);
        case ALV_CALL_ADJUST_LOGITS: return call(alv_adjust_logits, words, n);
        default: return fail(ALV_ERR_ARG, "no entry %d", entry);
    }
}
