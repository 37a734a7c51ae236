// err_flags.h -- what the device error flags mean, in plain C++ (tests/test_kv.py goes through all of them).
#pragma once

#include "../../include/hayai_cuda.h"

namespace hc {

constexpr int kErrRange = 1;    // an activation outside f16's range
constexpr int kErrWait = 2;     // a bounded wait ran out
constexpr int kErrKvRange = 4;  // a page number, length or offset out of range

struct ErrReport {
    int code;
    const char* text;
    // A block that gave up may have left its tiles' joining counters behind: they have to be cleared whatever
    // else was flagged, and is reported before it.
    bool clear_counters;
};
constexpr ErrReport err_report(int flag) {
    const bool clear = flag & kErrWait;
    if (flag & kErrRange)
        return {HC_ERR_RANGE, "an activation magnitude reached 65504 (outside the f16 range of the tensor-core split)", clear};
    if (flag & kErrWait) return {HC_ERR_TIMEOUT, "a bounded device wait expired", clear};
    if (flag & kErrKvRange)
        return {HC_ERR_INVALID, "kv batch: a page number, length or offset on the device is out of range", clear};
    return {HC_ERR_CUDA, "unknown device error flag", clear};
}

}  // namespace hc
