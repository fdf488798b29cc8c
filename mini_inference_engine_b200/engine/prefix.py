"""A prefix that requests share: tokens whose keys and values lie in the cache once (whole pages), for every request that begins with
them.  Made by ``LLMEngine.add_prefix``."""
from __future__ import annotations

import itertools

from ..cache.manager import RequestCache

_serials = itertools.count()


class Prefix:
    def __init__(self, token_ids):
        self.serial = next(_serials)
        self.token_ids = list(token_ids)     # of whole pages: what a request that shares it begins with
        self.cache = RequestCache()
        self.users = 0                       # requests that live and begin with it
        self.closed = False                  # released: its pages go back with the last user


def shared_groups(requests, block_size: int) -> list:
    """Rows of a step (requests in row order, those of a prefix side by side) as (rows, first row, shared positions) a group of rows that share pages."""
    out = []
    for i, s in enumerate(requests):
        key = (s.prefix.serial, s.cache.shared) if s.prefix is not None and s.cache.shared else None
        if key is not None and out and out[-1][0] == key and out[-1][2] + out[-1][1] == i:
            out[-1][1] += 1
        elif key is not None:
            out.append([key, 1, i])
    return [(n, first, key[1] * block_size) for key, n, first in out]
