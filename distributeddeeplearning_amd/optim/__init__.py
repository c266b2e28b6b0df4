from .fused import FusedSGD, FusedLARS, default_weight_decay_filter
from .muon import FusedMuon
from .lr import scaled_lr, staircase_multiplier, goyal_lr, poly_lr, LRSchedule
