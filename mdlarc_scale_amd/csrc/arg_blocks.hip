// The entries of K9 to K11 with their arguments in a block of memory.  A call through a foreign-function
// interface pays for each argument that it converts: a decode step's append (35 arguments) took Python
// 10.2 us with its checks, 9.2 so.
#include <string.h>

#include <cstddef>
#include <tuple>
#include <utility>

#include "mdlarc_hip.h"

namespace mdl {

namespace {

// the next argument of type A, at the next multiple of its alignment
template <typename A>
A take(const char* block, size_t& at) {
  at = (at + alignof(A) - 1) / alignof(A) * alignof(A);
  A a;
  memcpy(&a, block + at, sizeof(A));
  at += sizeof(A);
  return a;
}

template <typename... A, size_t... I>
int call(int (*entry)(A...), const void* block, void* stream, std::index_sequence<I...>) {
  if (!block) return MDL_ERR_NULL;
  using All = std::tuple<A...>;   // the stream is the last
  size_t at = 0;
  const std::tuple<std::tuple_element_t<I, All>...> args{
      take<std::tuple_element_t<I, All>>(static_cast<const char*>(block), at)...};   // in this order
  return entry(std::get<I>(args)..., stream);
}

template <typename... A>
int call(int (*entry)(A...), const void* block, void* stream) {
  return call(entry, block, stream, std::make_index_sequence<sizeof...(A) - 1>());
}

}  // namespace

}  // namespace mdl

extern "C" int mdl_rope_cache_paged_block(const void* args, void* stream) {
  return mdl::call(mdl_rope_cache_paged, args, stream);
}

extern "C" int mdl_paged_rows_block(const void* args, void* stream) {
  return mdl::call(mdl_paged_rows, args, stream);
}

extern "C" int mdl_attn_paged_block(const void* args, void* stream) {
  return mdl::call(mdl_attn_paged, args, stream);
}

extern "C" int mdl_sample_tokens_block(const void* args, void* stream) {
  return mdl::call(mdl_sample_tokens, args, stream);
}
