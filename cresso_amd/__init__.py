"""MI355X-native CRESSO5: the reference optimizer's per-step coordinate-field
hot path on hand-written gfx950 HIP kernels (libcresso_hip.so), and the
operators that make its gradients: embedding tables, the seams between blocks,
products with a frozen 8-bit weight, the distillation loss."""

from .blocks import block_product, quantize_blocks
from .distill import distill_loss, distill_loss_and_grad
from .embed import embedding, embedding_grad
from .optimizer import CRESSO, CRESSO5, count_optimizer_state_elements, theoretical_state_elements
from .seam import residual_norm

__all__ = ["CRESSO5", "CRESSO", "count_optimizer_state_elements", "theoretical_state_elements", "block_product",
           "quantize_blocks", "distill_loss", "distill_loss_and_grad", "embedding", "embedding_grad", "residual_norm"]
