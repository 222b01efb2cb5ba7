// A word that kernels set when a wait inside them ran out, and that the host takes back to 0 when it has told of it.
#pragma once

namespace fl {

struct FailedWord {
    int* word = nullptr;            // page-locked: a kernel's plain store is seen here
    bool take() { return word != nullptr && __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL) != 0; }
};

}  // namespace fl
