from .sampler import GenerationParams, Sampler, make_generator
from .scores import Candidate, ScoreBoard, TokenScore
