// Attention over the 4-bit cache instantiated for bf16 activations (see
// attn_mx4_impl.h).
#include "attn_mx4_impl.h"

namespace fxpr {
namespace attn {
namespace m4 {

int run_mx4_bf16(const Mx4Args& m, const Mx4Plan& p, int bits, int num_requests, int max_query_len, int64_t num_tokens,
             hipStream_t st) {
  switch (bits) {
    case 16: return dispatch_d<FXPR_DTYPE_BF16, 16>(m, p, num_requests, max_query_len, num_tokens, st);
    case 32: return dispatch_d<FXPR_DTYPE_BF16, 32>(m, p, num_requests, max_query_len, num_tokens, st);
    default: return dispatch_d<FXPR_DTYPE_BF16, 64>(m, p, num_requests, max_query_len, num_tokens, st);
  }
}

}  // namespace m4
}  // namespace attn
}  // namespace fxpr
