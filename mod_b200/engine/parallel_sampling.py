"""Several continuations of each prompt, sampled together.

1. each prompt is prefilled once;
2. it is forked into n sequences: their block tables share the prompt's full blocks, the partly filled last block is
   copied for each (one page-copy launch over all layers);
3. a step runs every sequence's last token and its n-gram drafts (``speculative.ngram_propose``) in one forward, whose
   attention reads the blocks of a common prompt once for all of its sequences (``attn_shared``);
4. the drafts are verified against the target's probabilities with given random numbers (``verify_sampled``): the
   emitted tokens follow the same distribution as sampling one token after another, greedy requests give the greedy
   tokens.  KV entries of refused drafts are overwritten later.

Where the blocks run out, the newest continuations give theirs back and come back later: forked again from the prompt, with
what they had emitted computed in one step before they go on.

On other backends than the native one the same steps run on the plain restatements of the operators.  Attention-only
models in a single process, as for n-gram speculation: recurrent state can neither be shared nor rolled back.
"""
from __future__ import annotations

import random
import time
from typing import Dict, List, Optional, Sequence as Seq, Tuple

import numpy as np
import torch

from ..ops import check_status
from .batch import ForwardBatch
from .sampler import filter_logits
from .sequence import SamplingParams, Sequence, SeqStatus
from .speculative import SpecStats, ngram_propose


class ParallelSampler:
    def __init__(self, engine, drafts: int = 4, ngram_max: int = 3, ngram_min: int = 1):
        if engine.runner.states is not None:
            raise ValueError("parallel sampling needs attention-only models (recurrent state cannot roll back)")
        if getattr(engine, "expert_parallel", False) or getattr(engine, "tensor_parallel", False):
            raise ValueError("parallel sampling runs in a single process")
        self.eng, self.k, self.nmax, self.nmin = engine, drafts, ngram_max, ngram_min
        self.native = getattr(engine.backend, "N", None) is not None and engine.device.type == "cuda"
        # on tensor cores a query group's head dim is 64, 128 or 256; elsewhere the prefill path serves
        self.shared = self.native and engine.cfg.head_dim in (64, 128, 256)
        self.stats = SpecStats()
        self.gen: Optional[torch.Generator] = None
        self.gens: Dict[int, Tuple[random.Random, torch.Generator]] = {}    # of seeded sequences, by request id

    # ------------------------------------------------------------------ random numbers
    def _seed(self, params: SamplingParams) -> None:
        self.gen = torch.Generator(device=self.eng.device)
        if params.seed is not None:
            self.gen.manual_seed(params.seed)
        else:
            self.gen.seed()

    def _draw(self, seqs: List[Sequence], K: int, V: int):
        """Uniforms [B, K] and Exp(1) noise [B, V].  Seeded sequences have generators of their own, which depend on the
        seed and on a sequence's place among its prompt's continuations, and draw as much in every step: what is emitted
        does not change with the other sequences.  It costs a launch a sequence (0.4 ms a step for 63 of 151936 ids)."""
        dev, B = self.eng.device, len(seqs)
        noise = torch.empty(B, V, device=dev)
        if not self.gens:
            return torch.rand(B, K, device=dev, generator=self.gen), noise.exponential_(generator=self.gen)
        rows = []
        for z, s in zip(noise, seqs):
            host, g = self.gens[s.req_id]
            rows.append([host.getrandbits(24) / 2 ** 24 for _ in range(max(1, self.k))][:K])
            z.exponential_(generator=g)
        return torch.tensor(rows).to(dev), noise

    # ------------------------------------------------------------------ verification
    def _verify(self, logits: torch.Tensor, counts: List[int], drafts: List[List[int]], seqs: List[Sequence]):
        """logits [sum(counts + 1), V] -> (accepted drafts, next token) of each sequence."""
        dev, B, K = logits.device, len(counts), max([1] + counts)
        ps = [s.params for s in seqs]
        heat = [max(p.temperature, 0.0) for p in ps]
        if any(t > 0 and (p.top_k > 0 or p.top_p < 1) for t, p in zip(heat, ps)):
            rows = [i for i, c in enumerate(counts) for _ in range(c + 1)]
            f = filter_logits(logits.float(), torch.tensor([heat[i] or 1.0 for i in rows], device=dev),
                              torch.tensor([ps[i].top_k for i in rows], device=dev),
                              torch.tensor([ps[i].top_p for i in rows], device=dev))
            sampled = torch.tensor([heat[i] > 0 for i in rows], device=dev)
            logits = torch.where(sampled[:, None], f, logits.float())   # filtered logits are already divided
            heat = [1.0 if t > 0 else 0.0 for t in heat]
        cu = torch.tensor(np.cumsum([0] + [c + 1 for c in counts]), dtype=torch.int32).to(dev)
        ids = torch.tensor([d + [0] * (K - len(d)) for d in drafts], dtype=torch.long).view(B, K).to(dev)
        uniforms, noise = self._draw(seqs, K, logits.shape[1])
        if self.native:
            ops = self.eng.backend.N
        else:
            from ..ops import reference as ops
        acc, tok, _ = ops.verify_sampled(logits.contiguous(), cu, ids, uniforms, noise,
                                         torch.tensor(heat, dtype=torch.float32).to(dev))
        acc, tok = torch.stack([acc.long(), tok]).tolist()
        if self.native:   # the step is over on the device: what a kernel gave up on is not emitted
            check_status(logits.device)
        if min(tok, default=0) < 0:
            raise RuntimeError("a row of logits has no finite entry")
        return acc, tok

    # ------------------------------------------------------------------ one step
    def _forward(self, seqs: List[Sequence], drafts: List[List[int]], groups: List[int], shared: List[int]):
        """Logits of every sequence's last token and drafts; ``groups``: sequences of each prompt (in order) and
        ``shared``: tokens whose blocks they have in common."""
        r = self.eng.runner
        bs, dev = r.blocks.block_size, r.device
        ids, pos, slots, ctx, qlens, rows = [], [], [], [], [], []
        bt = np.zeros((len(seqs), r.max_blocks), dtype=np.int32)
        for i, (s, d) in enumerate(zip(seqs, drafts)):
            start = s.num_cached      # the last emitted token is not cached yet, nor others after a time without blocks
            toks = s.output[start - len(s.prompt):] + d
            p = np.arange(start, start + len(toks))
            ids += toks
            pos.append(p)
            slots.append(np.asarray(s.blocks)[p // bs] * bs + p % bs)
            ctx.append(start + len(toks))
            qlens.append(len(toks))
            rows += range(len(ids) - 1 - len(d), len(ids))
            bt[i, :len(s.blocks)] = s.blocks

        def up(x, dtype=torch.int32):
            return torch.as_tensor(np.asarray(x)).to(dtype).to(dev)

        T = len(ids)
        fb = ForwardBatch(input_ids=up(ids, torch.long), positions=up(np.concatenate(pos)),
                          slot_mapping=up(np.concatenate(slots)), block_tables=torch.from_numpy(bt).to(dev),
                          ctx_lens=up(ctx), logits_idx=torch.arange(T, device=dev) if len(rows) == T else up(rows, torch.long),
                          state_slots=up([s.state_slot for s in seqs], torch.long), is_decode=False, query_lens=qlens,
                          ctx_lens_host=ctx)
        if self.shared:  # one schedule for all layers of the step
            m = r.model
            fb.shared_plan = self.eng.backend.N.attn_shared_plan(
                fb.block_tables, fb.ctx_lens, up(np.cumsum([0] + groups)), up(shared), T, m.Hq, m.Hkv,
                self.eng.cfg.head_dim, cu_q=up(np.cumsum([0] + qlens)))
        return r.model.logits(r.model.forward(fb, r.kv, r.states))

    def _make_room(self, seqs: List[Sequence]) -> None:
        """Blocks for everyone's last token; where they do not suffice, the newest sequences give theirs back."""
        eng = self.eng
        for s in seqs:
            while s.status == SeqStatus.RUNNING and not eng.blocks.allocate(s, s.length):
                running = [x for x in seqs if x.status == SeqStatus.RUNNING]
                if len(running) > 1:
                    eng.blocks.release(running[-1])
                    running[-1].status = SeqStatus.WAITING
                    eng.scheduler.num_preempted += 1
                elif eng.scheduler.running:    # other requests hold the rest
                    eng.step()
                else:
                    raise RuntimeError("KV cache exhausted during parallel sampling")

    def _most_blocks(self, s: Sequence) -> int:
        return self.eng.blocks.blocks_needed(max(s.length, len(s.prompt) + s.params.max_new_tokens - 1))

    def _resume(self, children: List[List[Sequence]]) -> None:
        """Forks sequences without blocks again, in order: while everyone who runs would still find all the blocks that
        it can come to need, so that none is computed anew more than once, and always one where nobody runs."""
        eng, m = self.eng, self.eng.blocks
        running = [c for cs in children for c in cs if c.status == SeqStatus.RUNNING]
        tokens = 0   # that are computed again in this step
        for cs in children:
            for c in cs:
                if c.status != SeqStatus.WAITING:
                    continue
                other = next((x for x in cs if x.status == SeqStatus.RUNNING), None)
                if running:
                    need = sum(self._most_blocks(x) - len(x.blocks) for x in running) + self._most_blocks(c)
                    need += 1 if other is None else -(len(c.prompt) // m.block_size)
                    if (need > m.num_free or len(m.free_slots) < 1 + (other is None)
                            or tokens + len(c.output) > eng.scheduler.max_prefill_tokens):
                        return
                if other is not None:
                    pairs = m.fork(other, c, len(c.prompt))
                    eng.kv.copy_pages(pairs)
                else:
                    self._fork_anew(c)
                c.status = SeqStatus.RUNNING
                running.append(c)
                tokens += len(c.output)

    def _fork_anew(self, c: Sequence) -> None:
        """The prompt of ``c`` once more, for it alone."""
        eng, parents = self.eng, []
        try:
            self._admit([c.prompt], 1, c.params, parents)
            p = parents[0]
            eng.runner.prefill([p], [p.length - p.num_cached], return_logits=True)
            if eng.prefix_caching:
                eng.blocks.register(p)
            eng.kv.copy_pages(eng.blocks.fork(p, c))
        finally:
            for p in parents:
                eng.blocks.release(p)

    def _step(self, running: List[List[Sequence]], shared: List[int]) -> None:
        eng = self.eng
        # everyone's last token first, drafts into what is left
        self._make_room([s for g in running for s in g])
        running = [[s for s in g if s.status == SeqStatus.RUNNING] for g in running]
        shared = [n for n, g in zip(shared, running) if g]
        running = [g for g in running if g]
        seqs = [s for g in running for s in g]
        drafts = []
        for s in seqs:
            room = min(self.k, s.params.max_new_tokens - len(s.output) - 1,
                       eng.runner.max_blocks * eng.blocks.block_size - s.length)
            d = ngram_propose(s.all_tokens, room, self.nmax, self.nmin) if room > 0 else []
            if d and not eng.blocks.allocate(s, s.length + len(d)):
                d = []
            drafts.append(d)
        logits = self._forward(seqs, drafts, [len(g) for g in running], shared)
        acc, tok = self._verify(logits, [len(d) for d in drafts], drafts, seqs)
        self.stats.steps += 1
        for s, d, a, t in zip(seqs, drafts, acc, tok):
            s.num_cached = s.length + a              # the last token and the accepted drafts
            self.stats.drafted += len(d)
            self.stats.accepted += a
            self._emit(s, d[:a] + [t])

    def _emit(self, s: Sequence, tokens: List[int]) -> None:
        n = 0
        for t in tokens:
            s.output.append(int(t))
            n += 1
            if s.finished_by(int(t)):
                s.status, s.t_finish = SeqStatus.FINISHED, time.perf_counter()
                self.eng.blocks.release(s)
                break
        self.stats.emitted += n
        self.stats.per_step.append(n)

    # ------------------------------------------------------------------ a wave of prompts
    def _admit(self, prompts: List[Seq[int]], n: int, params: SamplingParams, parents: List[Sequence]) -> None:
        """Gives blocks to the first prompts, as many as can be forked into n sequences each now, and appends them to
        ``parents``.  Where other requests hold what the first one needs, they are run until it is there."""
        eng, m = self.eng, self.eng.blocks
        forks = 0   # blocks that the forks will take: a copy of each partly filled last block
        for p in prompts:
            s = Sequence(prompt=[int(t) for t in p], params=params)
            more = n if s.length % m.block_size else 0

            def fits() -> bool:
                if not m.allocate(s, s.length):
                    return False
                if m.num_free >= forks + more and len(m.free_slots) >= n * (len(parents) + 1):
                    return True
                m.release(s)
                return False

            ok = fits()
            while not ok and not parents and eng.scheduler.running:
                eng.step()
                ok = fits()
            if not ok:
                if not parents:
                    raise RuntimeError(f"KV cache exhausted: a prompt of {s.length} tokens and its {n} continuations do not fit")
                return
            parents.append(s)
            forks += more

    def _wave(self, prompts: List[Seq[int]], n: int, params: SamplingParams) -> List[List[List[int]]]:
        """The continuations of the first prompts, of as many as there is room for."""
        eng, bs = self.eng, self.eng.blocks.block_size
        parents: List[Sequence] = []
        children: List[List[Sequence]] = []
        try:
            self._admit(prompts, n, params, parents)
            children += [[Sequence(prompt=list(p.prompt), params=params) for _ in range(n)] for p in parents]
            if params.seed is not None and params.temperature > 0:
                for cs in children:
                    for i, c in enumerate(cs):
                        host = random.Random(f"{params.seed} {i}")
                        self.gens[c.req_id] = host, torch.Generator(device=eng.device)
                        self.gens[c.req_id][1].manual_seed(host.getrandbits(63))
            rows, at = [], 0
            while at < len(parents):  # the prompts, as many at a time as a prefill step takes
                end, tokens = at, 0
                while end < len(parents) and (end == at or tokens + parents[end].length <= eng.scheduler.max_prefill_tokens):
                    tokens += parents[end].length - parents[end].num_cached
                    end += 1
                part = parents[at:end]
                rows.append(eng.runner.prefill(part, [p.length - p.num_cached for p in part], return_logits=True))
                at = end
            logits = torch.cat(rows)
            pairs = []
            for p, cs in zip(parents, children):
                if eng.prefix_caching:
                    eng.blocks.register(p)
                for c in cs:
                    c.status = SeqStatus.RUNNING
                    got = eng.blocks.fork(p, c)
                    if got is None:
                        raise RuntimeError("KV cache exhausted during parallel sampling")
                    pairs += got
            eng.kv.copy_pages(pairs)
            for p in parents:
                eng.blocks.release(p)
            every = [c for cs in children for c in cs]
            _, tok = self._verify(logits.repeat_interleave(n, 0), [0] * len(every), [[] for _ in every], every)
            for c, t in zip(every, tok):
                self._emit(c, [t])
            most = len(every)
            while True:
                self._resume(children)
                running = [[c for c in cs if c.status == SeqStatus.RUNNING] for cs in children]
                shared = [len(p.prompt) // bs * bs for p, g in zip(parents, running) if g]
                running = [g for g in running if g]
                if not running:
                    break
                left = sum(c.status != SeqStatus.FINISHED for c in every)
                # many have finished: their blocks lie between those that stay (with prefix caching too, but there a
                # compaction would give up the cached blocks of everyone's prompts)
                if 2 * left <= most and not eng.prefix_caching:
                    eng.compact_kv([c for g in running for c in g])
                    most = left
                self._step(running, shared)
            return [[c.output for c in cs] for cs in children]
        finally:
            for s in [*parents, *(c for cs in children for c in cs)]:
                if s.blocks or s.state_slot >= 0:
                    eng.blocks.release(s)
                self.gens.pop(s.req_id, None)

    def generate(self, prompts: List[Seq[int]], n: int, params: Optional[SamplingParams] = None) -> List[List[List[int]]]:
        """``n`` continuations of each prompt.  The prompts come in waves, each of as many as there are free blocks and
        places in the engine's batch to begin with; the continuations of a prompt begin together."""
        params = params or SamplingParams()
        if n < 1 or n >= self.eng.blocks.max_seqs:   # a slot for the prompt while it is forked
            raise ValueError(f"n = {n}: between 1 and {self.eng.blocks.max_seqs - 1} (the engine's batch less the prompt's)")
        if any(len(p) < 1 or len(p) + params.max_new_tokens > self.eng.runner.max_blocks * self.eng.blocks.block_size
               for p in prompts):
            raise ValueError("a prompt is empty or does not fit the model length with its new tokens")
        self._seed(params)
        out: List[List[List[int]]] = []
        while len(out) < len(prompts):
            out += self._wave(prompts[len(out):], n, params)
        return out
