from .plan import LayerSpec, ModelPlan, Run
from .model import Model
from .engine import Engine, EngineError, StepEntry
from .generate import generate, plan_batches, score, GenerationResult, GenerationStats, StepProfile, TokenScore

__all__ = ["LayerSpec", "ModelPlan", "Run", "Model", "Engine", "EngineError", "StepEntry", "generate",
           "plan_batches", "score", "GenerationResult", "GenerationStats", "StepProfile", "TokenScore"]
