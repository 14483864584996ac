// Small helpers of the operator layer (phase 1 checks and data pointers), shared by the files that define entry points.
#pragma once

#include <cstdint>
#include <initializer_list>

#include "internal.h"
#include "kernels.h"

namespace qmm {

inline int elem_type(aclDataType t) {
    switch (t) {
        case ACL_FLOAT: return ET_F32;
        case ACL_FLOAT16: return ET_F16;
        case ACL_BF16: return ET_BF16;
        case ACL_INT8: return ET_I8;
        case ACL_UINT8: return ET_U8;
        case ACL_INT4: return ET_I4;
        case ACL_INT32: return ET_I32;
        case ACL_FLOAT8_E4M3FN: return ET_E4M3;
        case ACL_FLOAT8_E5M2: return ET_E5M2;
        case ACL_FLOAT4_E2M1: return ET_E2M1;
        case ACL_FLOAT8_E8M0: return ET_E8M0;
        default: return ET_NONE;
    }
}
inline bool is_float_act(aclDataType t) { return t == ACL_FLOAT || t == ACL_FLOAT16 || t == ACL_BF16; }

inline const void *data_of(const aclTensor *t) {
    if (!t || !t->data) return nullptr;
    // Sub-byte tensors cannot carry an odd element offset; validated in phase 1.
    return (const char *)t->data + t->offset * (int64_t)elem_bits(elem_type(t->dtype)) / 8;
}

inline bool shape_is(const aclTensor *t, std::initializer_list<int64_t> dims) {
    if (t->viewDims.size() != dims.size()) return false;
    size_t i = 0;
    for (auto d : dims) if (t->viewDims[i++] != d) return false;
    return true;
}
inline bool dense(const aclTensor *t) { return t->contiguous(); }

// The code of a bounded wait that gave up on the current device, as last seen by aclnnB200DeviceStatus() (0: none).
uint32_t latched_status_of_current_device();

}  // namespace qmm
