"""Checkpoints by tensor name, their checks and the random-weights mode."""

from .adapters import AdapterError, pair_up, read_adapter, write_adapter
from .loader import (WeightError, cast, check, load_checkpoint, random_tensor, random_tensors,
                     write_model_folder)
from .safetensors_io import SafetensorsError, read_file, read_folder, write_file
from .spec import TensorSpec

__all__ = ["TensorSpec", "WeightError", "AdapterError", "SafetensorsError", "check", "cast", "load_checkpoint",
           "random_tensor", "random_tensors", "write_model_folder", "read_file", "read_folder", "write_file",
           "pair_up", "read_adapter", "write_adapter"]
