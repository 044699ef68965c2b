// gdn_once.cuh -- answers of the device that are asked for once (host code,
// plain C++).
#pragma once

#include <atomic>

namespace gdn {

// What `cell` holds, or else what ask() answers.  0 is no answer: a query that
// failed is asked again by the next call, whatever made it fail.  Host threads
// that ask at once get, and store, the same.
template <typename Ask>
int asked_once(std::atomic<int>& cell, Ask ask) {
    int v = cell.load();
    if (v == 0 && (v = ask()) != 0) cell.store(v);
    return v;
}

}  // namespace gdn
