"""B200-native TriangleMultiplication block (hand-written sm_100a kernels behind a C ABI).

Public surface:

* ``TriangleMultiplicationB200`` — ``nn.Module`` with the reference module's interface;
* ``triangle_multiplicative_update_b200`` — the reference's functional signature;
* ``BidirectionalTriangleMultiplicationB200`` / ``bidir_trimul_forward`` /
  ``bidirectional_triangle_multiplicative_update_b200`` — the reference's bidirectional block
  (outgoing and incoming contraction on the two halves of a doubled hidden width), as module, with
  this package's argument names and with those of the reference's functional op;
* ``install`` / ``from_reference`` — replace the reference's triangle-multiplication modules of an
  already-built model by their B200 twins (same parameters and ``state_dict`` keys);
* ``relative_position_bias_b200`` / ``RelativePositionBiasB200`` / ``PositionBuckets`` — the learned
  relative position bias by buckets, as the pair tensor's embedding and as an attention's bias, with
  the gradient of its table (``relative_position_bias_backward_b200``);
* ``cross_attention_b200`` — attention to states of another length with bias, padded keys and shared
  key heads, differentiable (``cross_attention_forward_b200`` / ``cross_attention_backward_b200``).

The compiled library ``libtrimul_b200.so`` is the only compute path; importing this
package does not load it, the first call does, and a missing library raises.
"""

from .functional import read_status, triangle_multiplicative_update_b200, trimul_forward, workspace_bytes
from .convert import from_reference, install
from .bidirectional import (BidirectionalTriangleMultiplicationB200, bidir_trimul_forward,
                            bidirectional_triangle_multiplicative_update_b200)
from .module import TriangleMultiplicationB200
from .relpos import (PositionBuckets, RelativePositionBiasB200, relative_position_bias_b200,
                     relative_position_bias_backward_b200)
from .attention import (AttentionState, cross_attention_b200, cross_attention_backward_b200,
                        cross_attention_forward_b200)

__all__ = [
    "TriangleMultiplicationB200",
    "BidirectionalTriangleMultiplicationB200",
    "bidir_trimul_forward",
    "bidirectional_triangle_multiplicative_update_b200",
    "install",
    "from_reference",
    "triangle_multiplicative_update_b200",
    "trimul_forward",
    "read_status",
    "workspace_bytes",
    "PositionBuckets",
    "RelativePositionBiasB200",
    "relative_position_bias_b200",
    "relative_position_bias_backward_b200",
    "AttentionState",
    "cross_attention_b200",
    "cross_attention_forward_b200",
    "cross_attention_backward_b200",
]
