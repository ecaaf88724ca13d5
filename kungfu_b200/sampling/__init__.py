from .sampler import CANDIDATES, RING, STATE_WORDS, Sampling, generator_state, pack_state
from .scores import MAX_ALTERNATIVES, ScoreRows, TokenScore, check_alternatives
