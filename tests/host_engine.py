"""``LLMEngine`` without a device: its requests, prefixes, grammars and steps, over a model that answers every request with the number of tokens that it has so far.  What a step
would launch is left out; everything that the host decides is the engine's own code."""
from mini_inference_engine_b200 import EngineConfig
from mini_inference_engine_b200.cache.manager import CacheManager, GroupSpec
from mini_inference_engine_b200.engine.engine import PENDING, LLMEngine, _InFlight
from mini_inference_engine_b200.engine.scheduler import Scheduler
from mini_inference_engine_b200.sampling.rules import RuleBook


class _Done:
    def synchronize(self):
        pass


class _Row(list):
    def tolist(self):
        return list(self)

    def __getitem__(self, at):
        return _Row(list.__getitem__(self, at))


class HostEngine(LLMEngine):
    def __init__(self, num_blocks, vocab=4096, eos=None, groups=None, **cfg):
        self.cfg = EngineConfig(num_blocks=num_blocks, **cfg)
        self.verbose, self.tokenizer, self.device = False, None, "cpu"
        self.eos_token_id, self.vocab_size = eos, vocab
        self.cache = CacheManager(groups or [GroupSpec("full")], num_blocks, self.cfg.block_size, 0)
        self.scheduler = Scheduler(self.cfg, self.cache)
        self.rules = RuleBook("cpu", self.cfg.max_model_len, vocab)
        self.can_share = self.cache.can_share()
        self.num_steps, self.ran, self.computed = 0, [], []       # ran: the requests of every step; computed: the prefixes' tokens
        self._host_state()

    def _compute_prefix(self, p):
        assert self.cache.reserve(p.cache, len(p.token_ids))
        self.cache.advance(p.cache, len(p.token_ids))
        self.computed.append(len(p.token_ids))

    def _launch(self):
        batch = self.scheduler.schedule()
        if not batch:
            return None
        last = [s for s, n in batch if s.cache.num_computed + n == len(s.token_ids)]
        tokens = _Row(len(s.token_ids) % self.vocab_size for s in last)
        self.ran.append([s.seq_id for s, _ in batch])
        ending = self._advance(batch, last)
        assert all(s.token_ids[-1] == PENDING for s in last)
        return _InFlight(last, [s.num_tokens - 1 for s in last], ending, [(tokens, len(last))], [(None, len(last))], _Done())
