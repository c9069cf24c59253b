from .adamw import AdamW
from .solver import CaffeSGD, build_optimizer
from .trainer import Trainer

__all__ = ["AdamW", "CaffeSGD", "build_optimizer", "Trainer"]
