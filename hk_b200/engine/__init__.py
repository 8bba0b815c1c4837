from .context import StepContext
from .engine import (BatchTooLarge, DeviceToken, Engine, EngineError, KernelTimeout, StepEntry, TokenOutOfRange, UnknownRequest, parse_dtype)
from .beams import BeamSearch, Continuation
from .drafts import DraftDecoder, LookupDrafts

__all__ = ["BatchTooLarge", "BeamSearch", "Continuation", "DeviceToken", "DraftDecoder", "Engine", "EngineError", "KernelTimeout", "LookupDrafts", "StepContext", "StepEntry", "TokenOutOfRange",
           "UnknownRequest", "parse_dtype"]
