"""The tests of shared prefixes once more, with groups taken at once however little they share."""
import pytest

from test_shared_prefix_gpu import *  # noqa: F401,F403
from test_shared_prefix_walk_gpu import at_once  # noqa: F401  (for every test)

pytestmark = pytest.mark.gpu
