from .engine import Engine, StepEntry, StepError
from .model import DecoderModel, expected_tensors
from .context import DraftEntry, EntryView, StepContext
from .generate import GenerateOutput, GenerateRequest, GenerationError, generate, plan_batches
from .api import BuiltEngine, EngineConfig, build

__all__ = ["Engine", "StepEntry", "DraftEntry", "StepError", "DecoderModel", "expected_tensors", "EntryView",
           "StepContext", "GenerateOutput", "GenerateRequest", "GenerationError", "generate",
           "plan_batches", "BuiltEngine", "EngineConfig", "build"]
