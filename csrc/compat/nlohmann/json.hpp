// torch's vmap headers include nlohmann/json.hpp, which torch does not ship,
// to write their interpreters out.  Nothing here does that: declarations are
// enough, and a call would not link.  Searched after every other include path,
// so a header that is there goes before this one.
#pragma once

#include <string>

namespace nlohmann {
struct json {
  json();
  template <typename T> json(const T&);
  static json parse(const std::string&);
  std::string dump() const;
  template <typename T> T get() const;
};
}  // namespace nlohmann
