// Host-side helpers shared by the sources of libovl_ssm.so.
#ifndef OVL_SSM_HOST_H_
#define OVL_SSM_HOST_H_

#include <stdint.h>
#include <string>

#include "ovl_ssm.h"

// ovl_status codes (ovl_launch.h)
#define OVL_SSM_OK 0
#define OVL_SSM_EHIP 4
#define OVL_SSM_EINVAL 6

namespace ovl_ssm {

int fail(int code, const std::string& detail);      // notes the text for ovl_ssm_last_error, returns the code
int after_launch(const char* who);                  // the HIP error of the launches since, if any

// HIP takes fewer than 2^32 work items in a launch.
inline bool launchable(uint64_t workgroups, uint64_t threads) { return workgroups <= 0xffffffffu / threads; }

inline uint64_t round_up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

}  // namespace ovl_ssm

#endif  // OVL_SSM_HOST_H_
