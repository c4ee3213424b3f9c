"""Module layer: the four classes python/featgraph/module/__init__.py:1-2 exports, plus
PartitionedSDDMMcuda (the reference's 2-D edge blocking on the GPU) and the operators that a
training step runs next to them (training.py)."""
from .spmm import SpMMbase, VanillaSpMMx86, VanillaSpMMcuda
from .sddmm import SDDMMbase, VanillaSDDMMx86, VanillaSDDMMcuda, PartitionedSDDMMcuda
from .training import EmbeddingLookupcuda, GradientClipcuda, SoftmaxCrossEntropycuda

__all__ = ["VanillaSpMMx86", "VanillaSpMMcuda", "VanillaSDDMMx86", "VanillaSDDMMcuda",
           "PartitionedSDDMMcuda", "SpMMbase", "SDDMMbase", "EmbeddingLookupcuda",
           "SoftmaxCrossEntropycuda", "GradientClipcuda"]
