from .batch import Segment, StepBatch, build_step_batch
from .executor import ContextOverflow, DraftTree, Engine, StepEntry, StepError
from ..kernels.api import KernelTimeout
from .model import Model, resolve_dtype

__all__ = ["Segment", "StepBatch", "build_step_batch", "ContextOverflow", "DraftTree", "Engine", "StepEntry",
           "StepError", "KernelTimeout", "Model", "resolve_dtype"]
