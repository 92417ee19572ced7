// The serving entries with their arguments as an array of 64-bit words.  A binding that converts
// its arguments one by one spends 3 us on 33 of them, more than the launch itself.
#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>

#include "cb_common.cuh"

namespace cb {
namespace {

template <typename A>
A from_word(int64_t word, bool& fits) {
  if constexpr (std::is_pointer<A>::value) {
    return reinterpret_cast<A>(static_cast<uintptr_t>(word));
  } else if constexpr (std::is_same<A, float>::value) {
    double value;
    memcpy(&value, &word, sizeof value);
    return static_cast<float>(value);
  } else {
    const A value = static_cast<A>(word);
    fits = fits && static_cast<int64_t>(value) == word;
    return value;
  }
}

template <typename... A, size_t... I>
int spread(int device, int (*entry)(A...), const int64_t* words, std::index_sequence<I...>) {
  bool fits = true;
  std::tuple<A...> args{from_word<A>(words[I], fits)...};
  CB_REQUIRE(fits, "an argument does not fit its type");
  const NullStreamDevice here(device);
  return entry(std::get<I>(args)...);
}

template <typename... A>
int unpack(int device, int (*entry)(A...), const int64_t* words, int64_t count) {
  CB_REQUIRE(count == static_cast<int64_t>(sizeof...(A)), "%lld words for %zu arguments", (long long)count, sizeof...(A));
  return spread(device, entry, words, std::index_sequence_for<A...>());
}

}  // namespace
}  // namespace cb

extern "C" int cb_call_packed(int entry, int device, const int64_t* words, int64_t num_words) {
  using namespace cb;
  clear_error();
  CB_REQUIRE(words != nullptr, "null pointer argument");
  CB_REQUIRE(device >= 0, "no device %d", device);
  switch (entry) {
    case CB_PACKED_APPEND_PAGED_KV:
      return unpack(device, cb_append_paged_kv, words, num_words);
    case CB_PACKED_APPEND_PAGED_KV4:
      return unpack(device, cb_append_paged_kv4, words, num_words);
    case CB_PACKED_GATHER_PAGED_KV4:
      return unpack(device, cb_gather_paged_kv4, words, num_words);
    case CB_PACKED_PAGED_ATTENTION4:
      return unpack(device, cb_paged_attention4, words, num_words);
    case CB_PACKED_PROMPT_ATTENTION:
      return unpack(device, cb_prompt_attention, words, num_words);
    default:
      set_error("no entry %d", entry);
      return CB_ERR_INVALID;
  }
}
