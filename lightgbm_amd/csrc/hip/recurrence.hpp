// Gated linear recurrence h[t] = a[t] h[t-1] + w[t] x[t] (w = 1, or 1 - a in the mixed form) and its gradients.
#pragma once
#include <cstdint>

namespace lga {

// Plain words only: the binding packs them one after the other.  Tensors are [batch][steps][width], neighbouring
// channels next to each other; *_b / *_t are the elements between sequences / steps.
struct ScanArgs {
  int64_t x, gate, state, lengths;    // gate, state, lengths: 0 = ones, zeros, all steps
  int64_t states, last;               // out (contiguous)
  int64_t work;                       // scan_workspace() bytes
  int64_t stream, device;
  int64_t batch, steps, width;
  int64_t x_b, x_t;
  int64_t gate_b, gate_t, groups;     // channel d takes the gate of group d / (width / groups)
  int64_t type, gate_type, mix;
};

struct ScanGradArgs {
  int64_t grad_states, states, gate, state, x, grad_last, lengths;   // state, x, grad_last, lengths may be 0
  int64_t grad_x, grad_state, grad_gate;                             // out (contiguous); grad_gate [gate_batch][steps][groups]
  int64_t work;                                                      // scan_grad_workspace() bytes
  int64_t stream, device;
  int64_t batch, steps, width;
  int64_t g_b, g_t, h_b, h_t, x_b, x_t;
  int64_t gate_b, gate_t, groups, gate_batch;
  int64_t type, gate_type, mix;
};

int64_t scan_workspace(const ScanArgs& a);
void gated_scan(const ScanArgs& a);
int64_t scan_grad_workspace(const ScanGradArgs& a);
void gated_scan_grad(const ScanGradArgs& a);

}  // namespace lga
