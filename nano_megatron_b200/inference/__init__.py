"""Checkpoint export to single-device artifacts, KV-cached and batched generation."""

from .artifact import (
    ARTIFACT_NAME,
    ARTIFACT_VERSION,
    InferenceArtifact,
    InferenceArtifactError,
    export_checkpoint,
    load_inference_artifact,
)
from .batch import BatchDecoder, LogitRules, generate_batch, generate_batch_from_artifact
from .generation import (
    GenerationResult,
    KVCacheDecoder,
    generate_from_artifact,
    generate_text,
    load_model_for_generation,
    sample_next_token,
)

__all__ = ["ARTIFACT_NAME", "ARTIFACT_VERSION", "BatchDecoder", "GenerationResult",
           "InferenceArtifact", "InferenceArtifactError", "KVCacheDecoder", "LogitRules",
           "export_checkpoint", "generate_batch", "generate_batch_from_artifact",
           "generate_from_artifact", "generate_text", "load_inference_artifact",
           "load_model_for_generation", "sample_next_token"]
