"""MI355X-native KGE score-function kernels behind the cuke apps/kge operator surface."""
from .kge import (KGEModel, TrainStep, Inspection, Forward, SparseGrads, inspect, inspector, margin_loss,
                  sparse_sgd, sparse_adagrad, transE, transH, transR, transF, RESCAL, KgeError)
from .data import KGDataset, TrainSampler
from .features import (FeatureEncoder, dropout, dropout_backward, linear, linear_backward, linear_forward,
                       preference_loss)

__all__ = ["KGEModel", "TrainStep", "Inspection", "Forward", "SparseGrads", "inspect", "inspector",
           "margin_loss", "sparse_sgd", "sparse_adagrad", "transE", "transH", "transR", "transF", "RESCAL",
           "KGDataset", "TrainSampler", "KgeError", "FeatureEncoder", "dropout", "dropout_backward", "linear",
           "linear_backward", "linear_forward", "preference_loss"]
