from .permutation import *  # noqa: F401,F403
from .few_tokens import *  # noqa: F401,F403
