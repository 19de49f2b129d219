// device_errors.h — the error codes that kernels record and the order in which the host is told.
#pragma once

namespace msst {

enum DeviceError : unsigned {
  kErrNone = 0,
  kErrTimeoutTmaFull = 1,
  kErrTimeoutSmemEmpty = 2,
  kErrTimeoutTmemFull = 3,
  kErrTimeoutTmemEmpty = 4,
  kErrTimeoutAttnS = 5,
  kErrTimeoutAttnP = 6,
  kErrTimeoutAttnO = 7,
  kErrTimeoutAttnQ = 8,
  kErrTimeoutAttnKV = 9,
  kErrTimeoutFfnS = 10,
  kErrTimeoutFfnP = 11,
  kErrTimeoutFfnO = 12,
  kErrTimeoutFfnFlag = 13,
  // not a wait: data of the call outside its documented range (see the operator)
  kErrPosition = 14,
  kErrAdapter = 15,
};

constexpr unsigned kFirstDataError = kErrPosition, kDataErrors = 2;

// What a translation unit's kernels have recorded: the first wait that gave up, and the data
// errors (bit i: kFirstDataError + i).
struct DeviceErrors {
  unsigned wait, data;
};

// Host: the code to report for n records, taken out of them: a wait that gave up before any data
// error (its results are garbage; all waits are taken out, as one leads to others), then the data
// errors one by one.  0: none.
inline unsigned take_error(DeviceErrors* e, int n) {
  unsigned wait = 0, data = 0;
  for (int i = 0; i < n; ++i) {
    if (!wait) wait = e[i].wait;
    e[i].wait = 0;
    data |= e[i].data;
  }
  if (wait) return wait;
  for (unsigned k = 0; k < kDataErrors; ++k) {
    if (!(data >> k & 1)) continue;
    for (int i = 0; i < n; ++i) e[i].data &= ~(1u << k);
    return kFirstDataError + k;
  }
  return 0;
}

}  // namespace msst
