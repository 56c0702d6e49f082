"""Operations on tensors: the interposed MPI_Allreduce, and the operators of a
language model (window attention, rotary positions, distillation)."""
from .allreduce import allreduce, allreduce_, mpi_datatype, mpi_op
from .attention import window_attention, window_attention_decode
from .distill import distill_loss
from .rotary import Rotary, rotary, rotary_

__all__ = ["allreduce", "allreduce_", "mpi_datatype", "mpi_op", "window_attention", "window_attention_decode",
           "Rotary", "rotary", "rotary_", "distill_loss"]
