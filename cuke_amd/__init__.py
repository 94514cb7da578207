"""MI355X-native KGE score-function kernels behind the cuke apps/kge operator surface."""
from .kge import (KGEModel, TrainStep, Inspection, Forward, SparseGrads, inspect, inspector, margin_loss,
                  sparse_sgd, sparse_adagrad, transE, transH, transR, transF, RESCAL, KgeError)
from .data import KGDataset, TrainSampler
from .features import (Block, FeatureEncoder, ResidualEncoder, Rows8, dropout, dropout_backward, linear, linear_backward,
                       linear_forward, pack8, preference_loss, rms_norm, rms_norm_backward, rms_norm_forward, unpack8)

__all__ = ["KGEModel", "TrainStep", "Inspection", "Forward", "SparseGrads", "inspect", "inspector",
           "margin_loss", "sparse_sgd", "sparse_adagrad", "transE", "transH", "transR", "transF", "RESCAL",
           "KGDataset", "TrainSampler", "KgeError", "FeatureEncoder", "dropout", "dropout_backward", "linear",
           "linear_backward", "linear_forward", "preference_loss", "Block", "ResidualEncoder", "Rows8", "pack8", "unpack8",
           "rms_norm", "rms_norm_backward", "rms_norm_forward"]
