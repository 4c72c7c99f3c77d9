"""MI355X-native DSA operator set (gfx950 HIP kernels behind a C ABI).

Public API, mirroring the reference's operator modules:

* ``sparse_flash_attention_triton`` / ``SparseFlashAttentionTriton``
* ``sparse_flash_attention_grad_triton`` / ``SparseFlashAttentionGradTriton``
* ``lightning_indexer_triton`` / ``LightningIndexerTriton``
* ``sparse_lightning_indexer_grad_kl_loss_triton`` /
  ``SparseLightningIndexerGradKLLossTriton``
* the dense warm-up stage: ``dense_lightning_indexer_softmax_lse_triton`` /
  ``DenseLightningIndexerSoftmaxLseTriton`` and ``dense_loss_backward_triton``
  / ``DenseLightningIndexerGradKLLossTriton`` (with their ``npu_`` aliases)

* around one decoding step: ``rotary_embedding`` / ``RotaryEmbedding``
  (with ``rotary_frequencies``), ``paged_cache_write`` / ``paged_cache_fork`` /
  ``paged_cache_compact``, and ``paged_attention`` / ``PagedAttention``
* for requests of many lengths: ``paged_cache_plan`` and
  ``paged_cache_write_slots``; for those that share a prefix:
  ``paged_cache_prefixes`` and ``paged_prefix_attention`` /
  ``PagedPrefixAttention``

and the autograd pairing for training (``autograd.py``):
``sparse_flash_attention_train`` / ``SparseFlashAttentionFunction`` and
``sparse_lightning_indexer_kl_loss`` / ``SparseLightningIndexerKLLossFunction``;
``rotary_embedding`` is differentiable itself (``RotaryEmbeddingFunction``).
"""
from .sparse_flash_attention import (  # noqa: F401
    INT64_MAX,
    SparseFlashAttentionTriton,
    sparse_flash_attention_triton,
)

from .sparse_flash_attention_grad import (  # noqa: F401
    SparseFlashAttentionGradTriton,
    sparse_flash_attention_grad_triton,
)

from .lightning_indexer import (  # noqa: F401
    LightningIndexerTriton,
    lightning_indexer_triton,
)

from .sparse_lightning_indexer_grad_kl_loss import (  # noqa: F401
    SparseLightningIndexerGradKLLossTriton,
    sparse_lightning_indexer_grad_kl_loss_triton,
)

from .dense_loss_backward import (  # noqa: F401
    DenseLightningIndexerGradKLLossTriton,
    DenseLightningIndexerSoftmaxLseTriton,
    DenseLossBackwardTriton,
    dense_lightning_indexer_grad_kl_loss_triton,
    dense_lightning_indexer_softmax_lse_triton,
    dense_loss_backward_triton,
    npu_dense_lightning_indexer_grad_kl_loss_triton,
    npu_dense_lightning_indexer_softmax_lse_triton,
)

from .rotary_embedding import (  # noqa: F401
    RotaryEmbedding,
    rotary_embedding,
    rotary_frequencies,
)

from .paged_cache import (  # noqa: F401
    paged_cache_compact,
    paged_cache_fork,
    paged_cache_plan,
    paged_cache_prefixes,
    paged_cache_write,
    paged_cache_write_slots,
)

from .paged_attention import (  # noqa: F401
    PagedAttention,
    PagedPrefixAttention,
    paged_attention,
    paged_prefix_attention,
)

sparse_flash_attention = sparse_flash_attention_triton
lightning_indexer = lightning_indexer_triton
sparse_flash_attention_grad = sparse_flash_attention_grad_triton
sparse_lightning_indexer_grad_kl_loss = sparse_lightning_indexer_grad_kl_loss_triton

from .autograd import (  # noqa: F401,E402
    RotaryEmbeddingFunction,
    SparseFlashAttentionFunction,
    SparseLightningIndexerKLLossFunction,
    sparse_flash_attention_train,
    sparse_lightning_indexer_kl_loss,
)
