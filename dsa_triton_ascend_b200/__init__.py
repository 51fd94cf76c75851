"""B200 (sm_100a) implementation of the DeepSeek Sparse Attention hot path.

Drop-in for the operators of 18851871668/dsa_triton_ascend, on CUDA torch tensors:

* :func:`sparse_flash_attention_triton` / :class:`SparseFlashAttentionTriton`
* :func:`sparse_flash_attention_grad_triton` / :class:`SparseFlashAttentionGradTriton`
* :func:`lightning_indexer_triton` / :class:`LightningIndexerTriton`
* :func:`sparse_lightning_indexer_grad_kl_loss_triton` /
  :class:`SparseLightningIndexerGradKLLossTriton`

plus :func:`sfa_fwd_bwd_from_host` (forward + backward of host-resident inputs, with the
copies overlapped with the kernels), :func:`lightning_indexer_paged` (the indexer over a
paged key cache, which the reference's indexer rejects), :func:`lightning_indexer_fp8` (the
FP8 indexer), the dense indexer KL loss of
:mod:`.dense_indexer_loss` (``dense_loss_backward_triton`` and its softmax-LSE helper) and
the autograd functions of :mod:`.autograd`.  For serving from a paged cache:
:func:`flash_attention_paged` (attention of new tokens over every cached key),
:func:`flash_attention_shared_prefix` (the same for rows that share their first pages),
:func:`rotary_embedding` and :func:`rotary_embedding_axes` (positions on several axes) with
:func:`rotary_table`, :func:`paged_cache_append`, :func:`paged_batch_plan` (a step's tables and slots from
its requests' lengths) with :func:`paged_cache_store`, and the upkeep
of the pages, :func:`paged_cache_extend`, :func:`paged_cache_fork`, :func:`paged_cache_free`,
:func:`paged_cache_compact` and :func:`paged_cache_copy`.
"""
from ._lib import check_device_errors, lib as _load_library  # noqa: F401
from .sparse_flash_attention import (  # noqa: F401
    SparseFlashAttentionTriton,
    sparse_flash_attention_triton,
)
from .lightning_indexer import (  # noqa: F401
    LightningIndexerTriton,
    lightning_indexer_fp8,
    lightning_indexer_paged,
    lightning_indexer_triton,
)
from .sparse_lightning_indexer_grad_kl_loss import (  # noqa: F401
    SparseLightningIndexerGradKLLossTriton,
    sparse_lightning_indexer_grad_kl_loss_partial,
    sparse_lightning_indexer_grad_kl_loss_triton,
)
from .sparse_flash_attention_grad import (  # noqa: F401
    SparseFlashAttentionGradTriton,
    sparse_flash_attention_grad_merged,
    sparse_flash_attention_grad_partial,
    sparse_flash_attention_grad_triton,
)
from .dense_indexer_loss import (  # noqa: F401
    DenseLightningIndexerGradKLLossTriton,
    DenseLightningIndexerSoftmaxLseTriton,
    DenseLossBackwardTriton,
    dense_lightning_indexer_grad_kl_loss_triton,
    dense_lightning_indexer_softmax_lse_triton,
    dense_loss_backward_triton,
    npu_dense_lightning_indexer_grad_kl_loss_triton,
    npu_dense_lightning_indexer_softmax_lse_triton,
)
from .flash_attention_paged import (  # noqa: F401
    flash_attention_paged,
    flash_attention_shared_prefix,
)
from .paged_cache import (  # noqa: F401
    PagedBatchPlan,
    paged_batch_plan,
    paged_cache_append,
    paged_cache_compact,
    paged_cache_copy,
    paged_cache_extend,
    paged_cache_fork,
    paged_cache_free,
    paged_cache_store,
)
from .rotary_embedding import (  # noqa: F401
    rotary_axes,
    rotary_embedding,
    rotary_embedding_axes,
    rotary_frequencies,
    rotary_table,
)
from .streaming import bind_host_to_device, host_outputs, sfa_fwd_bwd_from_host  # noqa: F401
from .autograd import (  # noqa: F401
    IndexerKLLossFunction,
    RotaryEmbeddingAxesFunction,
    RotaryEmbeddingFunction,
    SparseAttentionWithIndexer,
    SparseFlashAttentionFunction,
)

__all__ = [
    "sparse_flash_attention_triton",
    "SparseFlashAttentionTriton",
    "sparse_flash_attention_grad_triton",
    "SparseFlashAttentionGradTriton",
    "lightning_indexer_triton",
    "LightningIndexerTriton",
    "sparse_lightning_indexer_grad_kl_loss_triton",
    "SparseLightningIndexerGradKLLossTriton",
    "flash_attention_paged",
    "flash_attention_shared_prefix",
    "rotary_embedding",
    "rotary_embedding_axes",
    "rotary_axes",
    "rotary_table",
    "PagedBatchPlan",
    "paged_batch_plan",
    "paged_cache_append",
    "paged_cache_compact",
    "paged_cache_copy",
    "paged_cache_extend",
    "paged_cache_fork",
    "paged_cache_free",
    "paged_cache_store",
    "check_device_errors",
]
