"""Op layer: the ten names python/featgraph/op/__init__.py:1-5 exports, and the training
operators that stand next to them."""
from .vanilla_spmm import (vanilla_spmm_csr_cuda, schedule_vanilla_spmm_csr_cuda,
                           vanilla_spmm_csr_x86, schedule_vanilla_spmm_csr_x86,
                           vanilla_spmm_dds_x86, schedule_vanilla_spmm_dds_x86)
from .vanilla_sddmm import (vanilla_sddmm, schedule_vanilla_sddmm_cuda_tree_reduce,
                            schedule_vanilla_sddmm_cuda_single_thread_reduce,
                            schedule_vanilla_sddmm_x86)
from .training import (embedding_lookup, schedule_embedding_lookup_cuda,
                       softmax_cross_entropy, schedule_softmax_cross_entropy_cuda,
                       gradient_clip, schedule_gradient_clip_cuda)

__all__ = [
    "vanilla_spmm_csr_cuda", "schedule_vanilla_spmm_csr_cuda",
    "vanilla_spmm_csr_x86", "schedule_vanilla_spmm_csr_x86",
    "vanilla_spmm_dds_x86", "schedule_vanilla_spmm_dds_x86",
    "vanilla_sddmm", "schedule_vanilla_sddmm_cuda_tree_reduce",
    "schedule_vanilla_sddmm_cuda_single_thread_reduce", "schedule_vanilla_sddmm_x86",
    "embedding_lookup", "schedule_embedding_lookup_cuda",
    "softmax_cross_entropy", "schedule_softmax_cross_entropy_cuda",
    "gradient_clip", "schedule_gradient_clip_cuda",
]
