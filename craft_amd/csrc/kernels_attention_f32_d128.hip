// float attention, head width up to 128 (attention_fwd / _token / _bwd.inc.hpp)
#include "attention_fwd.inc.hpp"
#include "attention_token.inc.hpp"
#include "attention_bwd.inc.hpp"
namespace craft {
template int attention_fwd_launch<float, 128>(const AttentionParams&, hipStream_t);
template int attention_token_launch<float, 128>(const AttentionParams&, hipStream_t);
template int attention_bwd_launch<float, 128>(const AttentionParams&, hipStream_t);
}  // namespace craft
