// The balance loss's passes over the rows, __bf16 scores.
#include "losses_balance.hpp"

namespace wgbm {

int balance_stats_bf16(const ScoresView& s, const uint8_t* mask, int32_t top_k, const BalanceWs& w,
                     int32_t* slots, hipStream_t st) {
  return balance_stats<__bf16>(s, mask, top_k, w, slots, st);
}

int balance_grad_bf16(const ScoresView& s, const BalanceWs& w, const ScoresView& out,
                    bool accumulate, hipStream_t st) {
  return balance_grad<__bf16>(s, w, out, accumulate, st);
}

}  // namespace wgbm
