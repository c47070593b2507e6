// sequence_attention_back.hip -- the walk backwards in time, for the gradients of k, v and the state (a translation unit of its own:
// the two directions compile side by side).
#include "sequence_walk.h"

namespace fishing {
namespace seq {

template int walk<float, true>(const FishingDecayAttention*, Strided, Strided, Strided, const float*, float*, Strided, int, int, bool, bool, double, double, Shared*, void*, hipStream_t);
template int walk<bf16, true>(const FishingDecayAttention*, Strided, Strided, Strided, const float*, float*, Strided, int, int, bool, bool, double, double, Shared*, void*, hipStream_t);

}  // namespace seq
}  // namespace fishing
