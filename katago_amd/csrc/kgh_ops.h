// Launchers and checks of the operators on the caller's tensors (katago_hip.h),
// and the device code that they share.
#ifndef KGH_OPS_H
#define KGH_OPS_H

#include "kgh_common.h"

#include "../../include/katago_hip.h"

typedef __bf16 bf16_t;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

namespace kgh {

// The calling thread's current device, put back at the end of the scope.
struct DeviceScope {
  int before = -1;
  bool changed = false;
  explicit DeviceScope(int device);
  ~DeviceScope();
};

// pointers: whether the params' pointers are looked at too.
void checkLinear(const kgh_linear_params& p, bool pointers);
uint64_t linearWorkspace(const kgh_linear_params& p);
void launchLinear(const kgh_linear_params& p, hipStream_t stream);

void checkRope(const kgh_rope_params& p);
void launchRope(const kgh_rope_params& p, hipStream_t stream);

void checkAttention(const kgh_attention_params& p, bool pointers);
uint64_t attentionWorkspace(const kgh_attention_params& p);
void launchAttention(const kgh_attention_params& p, hipStream_t stream);

void checkQuantize(const kgh_quantize_params& p);
void launchQuantize(const kgh_quantize_params& p, hipStream_t stream);

void checkLinearInt8(const kgh_linear_int8_params& p, bool pointers);
uint64_t linearInt8Workspace(const kgh_linear_int8_params& p);
void launchLinearInt8(const kgh_linear_int8_params& p, hipStream_t stream);

void checkGroupNorm(const kgh_group_norm_params& p, bool pointers);
uint64_t groupNormWorkspace(const kgh_group_norm_params& p);
void launchGroupNorm(const kgh_group_norm_params& p, hipStream_t stream);

void checkGroupNormBackward(const kgh_group_norm_backward_params& p, bool pointers);
uint64_t groupNormBackwardWorkspace(const kgh_group_norm_backward_params& p);
void launchGroupNormBackward(const kgh_group_norm_backward_params& p, hipStream_t stream);

inline void opInvalid(const char* op, const std::string& m) { throw KghError(KGH_ERR_INVALID_ARGUMENT, std::string(op) + ": " + m); }
inline size_t opElemBytes(int dtype) { return dtype == KGH_DTYPE_FP32 ? 4 : 2; }
inline void opCheckDtype(const char* op, int dtype) {
  if(dtype != KGH_DTYPE_FP32 && dtype != KGH_DTYPE_FP16 && dtype != KGH_DTYPE_BF16)
    opInvalid(op, "dtype " + std::to_string(dtype) + " is none of KGH_DTYPE_*");
}
inline void opCheckActivation(const char* op, int act) {
  if(act != KGH_ACTIVATION_IDENTITY && act != KGH_ACTIVATION_RELU && act != KGH_ACTIVATION_MISH && act != KGH_ACTIVATION_SILU && act != KGH_ACTIVATION_GELU)
    opInvalid(op, "activation " + std::to_string(act) + " is none of KGH_ACTIVATION_*");
}
// A tensor's pointer: present, and aligned to its elements.
inline void opCheckPointer(const char* op, const char* name, const void* p, size_t elem) {
  if(p == nullptr) opInvalid(op, std::string(name) + " is null");
  if((uintptr_t)p % elem != 0) opInvalid(op, std::string(name) + " is not aligned to its elements");
}
// An input that the output must not overlap.
inline void opCheckApart(const char* op, const char* name, const void* in, const void* out) {
  if(in == out) opInvalid(op, std::string("out is ") + name + " itself");
}
// A workspace that a call cannot do without.
inline void opCheckWorkspace(const char* op, const void* workspace, uint64_t bytes, uint64_t need) {
  if(workspace != nullptr) opCheckPointer(op, "workspace", workspace, 16);
  if(need > 0 && (workspace == nullptr || bytes < need))
    opInvalid(op, "needs a workspace of " + std::to_string(need) + " bytes, has " + std::to_string(workspace == nullptr ? 0 : bytes));
}
// Calls f(T()) for the element type of dtype.
template<typename F>
void withDtype(int dtype, F&& f) {
  if(dtype == KGH_DTYPE_FP32) f(float());
  else if(dtype == KGH_DTYPE_FP16) f(half_t());
  else f(bf16_t());
}

}  // namespace kgh

#endif
