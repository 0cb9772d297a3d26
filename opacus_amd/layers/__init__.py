from .dp_multihead_attention import DPMultiheadAttention, SequenceBias
from .dp_rnn import DPGRU, DPLSTM, DPRNN, RNNLinear
from .gated_rnn import DPGatedRNN, GatedScan
from .norm_act import GroupNormAct, HeadNormAct
from .param_rename import RenameParamsMixin

__all__ = [
    "DPRNN",
    "DPGRU",
    "DPLSTM",
    "DPGatedRNN",
    "DPMultiheadAttention",
    "GatedScan",
    "GroupNormAct",
    "HeadNormAct",
    "RNNLinear",
    "RenameParamsMixin",
    "SequenceBias",
]
