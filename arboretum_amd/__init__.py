"""MI355X-native histogram tree growing behind arboretum's C-ABI and Python API."""
from .core import (ArboretumClassifier, ArboretumError, ArboretumRegression, DMatrix, Garden,
                   adamw, copy_probe, device_count, embedding, embedding_grad, embedding_grad_bytes,
                   embedding_sort, embedding_sort_bytes, hist_sum, hist_sum_no_alloc, hist_sum_plan, load, release_memory,
                   train)

__all__ = ["DMatrix", "Garden", "train", "load", "ArboretumRegression", "ArboretumClassifier",
           "ArboretumError", "device_count", "hist_sum", "hist_sum_no_alloc", "hist_sum_plan", "release_memory",
           "embedding", "embedding_sort", "embedding_sort_bytes", "embedding_grad", "embedding_grad_bytes", "adamw"]
