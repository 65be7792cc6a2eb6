// Rules on a batch of logits: launches of logits.hip.
#pragma once

#include "tla_internal.h"

namespace tla {

// Words from one row's arrival counter to the next: device-scope atomics on one
// line of memory wait for each other (0.11 us each).
constexpr int kRowCounterStride = 64;

struct LogitsParams {
    const float* x;  // [n_seq][n_vocab]
    float* out;      // may be x
    int* tokens;     // [n_seq], or NULL
    int n_vocab;
    int slice;       // logits per workgroup (logits_slice)
    int n_slices;    // workgroups per row
    tla_logit_rules rules;
    // With tokens and several slices: each workgroup's best (an argmax key),
    // [n_seq][n_slices], and the rows' arrivals, kRowCounterStride apart; zero between launches.
    unsigned long long* best;
    int* counters;
};

// Logits per workgroup.
int logits_slice(int n_seq, int n_vocab, int n_cu);
hipError_t launch_logits_process(const LogitsParams& p, int n_seq, hipStream_t s);
hipError_t load_logits_code();

}  // namespace tla
