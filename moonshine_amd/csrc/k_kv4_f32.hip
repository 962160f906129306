// Attention over the 4-bit cache for f32 queries (kv4_attention.h).
#include "kv4_attention.h"

namespace msh {
void kv4_attention_f32(const Kv4Attention& a, hipStream_t s) { dispatch_kv4_attention<Elem::f32>(a, s); }
}  // namespace msh
