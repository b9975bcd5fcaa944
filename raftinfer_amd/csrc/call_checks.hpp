// Host checks that the entry points of several operators share.
#pragma once

#include "common.hpp"

#include <initializer_list>

namespace raftinfer::amd {

// The stream's device for the launches of a call, where another one is current.
template <typename Error> class StreamDevice {
public:
  StreamDevice(hipStream_t stream, const char *caller) {
    int device = 0;
    if (hipGetDevice(&current_) != hipSuccess || hipStreamGetDevice(stream, &device) != hipSuccess)
      throw Error(std::string{caller} + " HIP stream has no device");
    if (device == current_) return;
    if (hipSetDevice(device) != hipSuccess) throw Error(std::string{caller} + " cannot select the stream's device");
    changed_ = true;
  }
  ~StreamDevice() {
    if (changed_) (void)hipSetDevice(current_);
  }
  StreamDevice(const StreamDevice &) = delete;
  StreamDevice &operator=(const StreamDevice &) = delete;

private:
  int current_ = 0;
  bool changed_ = false;
};

inline bool aligned16(const void *p) { return (reinterpret_cast<std::uintptr_t>(p) & 15u) == 0; }

// Whether no two vectors of `width` elements, n0 by n1 of them with strides s0 and s1, share an
// element (told for strides of which one steps over all of the other's).
inline bool strides_apart(std::size_t n0, std::size_t s0, std::size_t n1, std::size_t s1, std::size_t width) {
  const auto over = [&](std::size_t inner_n, std::size_t inner, std::size_t outer_n, std::size_t outer) {
    return (inner_n == 1 || inner >= width) && (outer_n == 1 || outer >= (inner_n - 1) * inner + width);
  };
  return over(n1, s1, n0, s0) || over(n0, s0, n1, s1);
}

struct Bytes {
  const void *at;
  std::size_t count;
};
// What a call writes overlaps neither what it reads nor what else it writes.
template <typename Error>
inline void validate_apart(std::initializer_list<Bytes> written, std::initializer_list<Bytes> read, const char *message) {
  const auto apart = [](const Bytes &a, const Bytes &b) {
    const auto x = reinterpret_cast<std::uintptr_t>(a.at), y = reinterpret_cast<std::uintptr_t>(b.at);
    return a.count == 0 || b.count == 0 || (x <= y ? a.count <= y - x : b.count <= x - y);
  };
  for (auto w = written.begin(); w != written.end(); ++w) {
    for (auto other = w + 1; other != written.end(); ++other) require<Error>(apart(*w, *other), message);
    for (const Bytes &r : read) require<Error>(apart(*w, r), message);
  }
}

} // namespace raftinfer::amd
