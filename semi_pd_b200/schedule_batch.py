"""Request / batch bookkeeping the schedulers use to build `ModelWorkerBatch`es — the slice of
python/sglang/srt/managers/schedule_batch.py the semi-PD path exercises:
`Req` (:246-513), `ScheduleBatch.prepare_for_extend` (:790-985, incl. the
`pre_allocated_req_pool_indices` variant the prefill worker uses, :923-935),
`prepare_for_decode` (:1144-1207), `filter_batch` / `merge_batch` (:1209-1306),
`check_decode_mem` / `retract_decode` (:1022-1125) and `get_model_worker_batch` (:1308-1370).
Sampling is greedy-only; logprobs / grammar / multimodal are off this path
(managers/semi_pd_scheduler.py:207-209, semi_pd_decode_scheduler.py:354).
"""
from __future__ import annotations

import copy
import dataclasses
from typing import List, Optional, Sequence

import torch

from . import ops
from .forward_batch_info import ForwardMode, ModelWorkerBatch, SharedPrefix
from .memory_pool import ReqToTokenPool, TokenToKVPoolAllocator, compact_request, fork_request

_bid = 0


@dataclasses.dataclass
class SamplingParams:
    max_new_tokens: int = 128
    ignore_eos: bool = True
    temperature: float = 0.0  # greedy


class Req:
    """The input and output status of a request."""

    def __init__(self, rid: str, origin_input_ids: List[int], sampling_params: SamplingParams,
                 eos_token_ids: Optional[set] = None, arrival_time: float = 0.0):
        self.rid = rid
        self.origin_input_ids = list(origin_input_ids)
        self.output_ids: List[int] = []
        self.fill_ids: List[int] = []
        self.sampling_params = sampling_params
        self.eos_token_ids = eos_token_ids or set()
        self.req_pool_idx: Optional[int] = None
        self.prefix_indices: List[int] = []   # length = tokens already in the KV pool
        self.extend_input_len = 0
        self.is_chunked = 0
        self.is_retracted = False
        self.finished_reason: Optional[str] = None
        # tokens whose computation has been launched (>= len(output_ids) under the overlap loop)
        self.launched_tokens = 0
        # tokens that compactions took out of the cache: the next one's position is that many ahead of the cache's length
        self.dropped_tokens = 0
        self.num_forks = 0   # continuations forked off (their rids are numbered)
        # timing (host clock, seconds)
        self.arrival_time = arrival_time
        self.first_token_time: Optional[float] = None
        self.finish_time: Optional[float] = None
        self.token_times: List[float] = []
        # output / timestamps produced before a retraction (this Req then continues the request
        # with prompt + those tokens as its input; stitched back together when it finishes)
        self.prior_output_ids: List[int] = []
        self.prior_token_times: List[float] = []
        self.retracted_from: Optional["Req"] = None

    @property
    def seqlen(self):
        return len(self.origin_input_ids) + len(self.output_ids)

    def finished(self) -> bool:
        return self.finished_reason is not None

    def init_next_round_input(self, prefix_len: Optional[int] = None):
        self.fill_ids = self.origin_input_ids + self.output_ids
        if prefix_len is not None:
            self.prefix_indices = [0] * prefix_len  # only the length matters (no radix cache)
        self.extend_input_len = len(self.fill_ids) - len(self.prefix_indices)

    def check_finished(self):
        if self.finished():
            return
        if len(self.output_ids) >= self.sampling_params.max_new_tokens:
            self.finished_reason = "length"
            return
        if not self.sampling_params.ignore_eos and self.output_ids and \
                self.output_ids[-1] in self.eos_token_ids:
            self.finished_reason = "stop"

    def reset_for_retract(self):
        self.prefix_indices = []
        self.extend_input_len = 0
        self.is_retracted = True
        self.req_pool_idx = None
        self.dropped_tokens = 0


class ScheduleBatch:
    """Store all information of a batch on the scheduler."""

    def __init__(self, reqs: List[Req], req_to_token_pool: ReqToTokenPool,
                 token_to_kv_pool_allocator: TokenToKVPoolAllocator, device):
        self.reqs = reqs
        self.req_to_token_pool = req_to_token_pool
        self.token_to_kv_pool_allocator = token_to_kv_pool_allocator
        self.device = device
        self.forward_mode: Optional[ForwardMode] = None
        self.input_ids = None
        self.req_pool_indices = None
        self.seq_lens = None
        self.out_cache_loc = None
        self.output_ids = None
        self.seq_lens_sum = 0
        self.seq_lens_host: List[int] = []   # host mirror of `seq_lens` (the run allocator's view)
        self.prefix_lens = None
        self.extend_lens = None
        self.extend_num_tokens = None
        self.decoding_reqs = None
        self._shared = None   # (groups of the last step, SharedPrefix, its lists)
        self._compacted = False   # some request may have dropped tokens

    @classmethod
    def init_new(cls, reqs, req_to_token_pool, token_to_kv_pool_allocator, device=None):
        return cls(reqs, req_to_token_pool, token_to_kv_pool_allocator,
                   device or req_to_token_pool.device)

    def batch_size(self):
        return len(self.reqs)

    def is_empty(self):
        return len(self.reqs) == 0

    # --- allocation -----------------------------------------------------------------------------
    def alloc_req_slots(self, num_reqs: int):
        idx = self.req_to_token_pool.alloc(num_reqs)
        if idx is None:
            raise RuntimeError("alloc_req_slots runs out of memory. Please set a smaller number for "
                               "`--max-running-requests`.")
        return idx

    def _oom(self, phase: str, num_tokens: int):
        return RuntimeError(f"{phase} out of memory. Try to lower your batch size. "
                            f"Try to allocate {num_tokens} tokens; available "
                            f"{self.token_to_kv_pool_allocator.available_size()}.")

    def _h2d(self, values, dtype):
        return torch.tensor(values, dtype=dtype, pin_memory=True).to(self.device, non_blocking=True)

    # --- extend ---------------------------------------------------------------------------------
    def prepare_for_extend(self, pre_allocated_req_pool_indices: Optional[List[int]] = None):
        """Decode-side call (pre_allocated None): allocates request + KV slots and writes
        req_to_token.  Prefill-side call: adopts the request slots the decode side chose and reads
        out_cache_loc back from the shared req_to_token table (schedule_batch.py:923-935)."""
        self.forward_mode = ForwardMode.EXTEND
        bs = len(self.reqs)
        reqs = self.reqs
        if any(r.dropped_tokens for r in reqs):
            raise NotImplementedError("a request whose cache was compacted takes no further prompt tokens")
        input_ids = [r.fill_ids[len(r.prefix_indices):] for r in reqs]
        extend_num_tokens = sum(len(ids) for ids in input_ids)
        seq_lens = [len(r.fill_ids) for r in reqs]
        prefix_lens = [len(r.prefix_indices) for r in reqs]
        extend_lens = [r.extend_input_len for r in reqs]

        if pre_allocated_req_pool_indices is None:
            # a chunked / continued request keeps its slot
            need = [r for r in reqs if r.req_pool_idx is None]
            new_idx = self.alloc_req_slots(len(need))
            for r, i in zip(need, new_idx):
                r.req_pool_idx = i
            req_pool_indices = [r.req_pool_idx for r in reqs]
        else:
            req_pool_indices = list(pre_allocated_req_pool_indices)
            for r, i in zip(reqs, req_pool_indices):
                r.req_pool_idx = i

        if all(getattr(r, "input_ids_device", None) is not None for r in reqs):
            # prompt ids already resident in HBM (bench.py's device-resident arm): slice, no H2D
            parts = [r.input_ids_device[len(r.prefix_indices):len(r.fill_ids)] for r in reqs]
            self.input_ids = parts[0] if len(parts) == 1 else torch.cat(parts)
        else:
            self.input_ids = self._h2d([t for ids in input_ids for t in ids], torch.int64)
        self.req_pool_indices = self._h2d(req_pool_indices, torch.int64)
        self.seq_lens = self._h2d(seq_lens, torch.int64)
        prefix_lens_t = self._h2d(prefix_lens, torch.int64)
        extend_lens_t = self._h2d(extend_lens, torch.int64)

        if pre_allocated_req_pool_indices is None:
            # runs: positions [pre, seq) of every request continue its last run, then take whole
            # new runs (memory_pool.TokenToKVPoolAllocator.alloc_extend)
            self.out_cache_loc = self.token_to_kv_pool_allocator.alloc_extend(
                req_pool_indices, prefix_lens, seq_lens)
            if self.out_cache_loc is None:
                raise self._oom("Prefill", extend_num_tokens)
            ops.write_req_to_token_pool(self.req_to_token_pool.req_to_token, self.req_pool_indices,
                                        prefix_lens_t, self.seq_lens, extend_lens_t,
                                        self.out_cache_loc)
        else:
            # gather out_cache_loc = req_to_token[req, pre:seq] on the device (no host sync)
            kv_indptr = self._h2d([0] + list(_cumsum(extend_lens)), torch.int32)
            loc32 = torch.empty((extend_num_tokens,), dtype=torch.int32, device=self.device)
            ops.create_kv_indices(self.req_to_token_pool.req_to_token, self.req_pool_indices,
                                  extend_lens_t.int(), kv_indptr, prefix_lens_t.int(), loc32)
            self.out_cache_loc = loc32.long()

        self.seq_lens_sum = sum(seq_lens)
        self.seq_lens_host = list(seq_lens)
        self.extend_num_tokens = extend_num_tokens
        self.prefix_lens = prefix_lens
        self.extend_lens = extend_lens

    # --- decode ---------------------------------------------------------------------------------
    def check_decode_mem(self, buf_multiplier: int = 1) -> bool:
        """Can every request of the batch get the slot of its next token?  Exact under the run
        allocator: only requests whose last run is full need a new one."""
        return self.token_to_kv_pool_allocator.can_alloc_decode(self.seq_lens_host)

    def retract_decode(self, retract_decode_steps: int = 20):
        """Retract requests with the fewest generated tokens / longest prompts first until
        `retract_decode_steps` slots per remaining request are free (schedule_batch.py:1034-1111)."""
        order = sorted(range(len(self.reqs)),
                       key=lambda i: (len(self.reqs[i].output_ids), -len(self.reqs[i].origin_input_ids)),
                       reverse=True)
        retracted = []
        alloc = self.token_to_kv_pool_allocator
        while (alloc.available_size() < alloc.ceil_to_run(len(order) * retract_decode_steps)
               and len(order) > 1):
            idx = order.pop()
            req = self.reqs[idx]
            retracted.append(req)
            alloc.free_req(req.req_pool_idx)
            self.req_to_token_pool.free(req.req_pool_idx)
            req.reset_for_retract()
        self.filter_batch(keep_indices=sorted(order))
        return retracted

    def prepare_for_decode(self):
        self.forward_mode = ForwardMode.DECODE
        bs = len(self.reqs)
        # the token sampled by the previous step is this step's input
        self.input_ids = self.output_ids
        self.output_ids = None
        self.out_cache_loc = self.token_to_kv_pool_allocator.alloc_decode(
            [r.req_pool_idx for r in self.reqs], self.seq_lens_host)
        if self.out_cache_loc is None:
            raise self._oom("Decode", bs)
        # req_to_token[req, seq_len] = slot ; seq_lens += 1   (schedule_batch.py:1186-1207)
        ops.write_req_to_token_pool(self.req_to_token_pool.req_to_token, self.req_pool_indices,
                                    self.seq_lens, self.seq_lens + 1,
                                    torch.ones_like(self.seq_lens), self.out_cache_loc)
        self.seq_lens = self.seq_lens + 1
        self.seq_lens_host = [s + 1 for s in self.seq_lens_host]
        self.seq_lens_sum += bs

    def fork_req(self, index: int, n: int) -> Optional[List[Req]]:
        """n more continuations of request `index` of a decode batch, between two steps: requests like it (prompt and output
        so far) right behind it in the batch, so that neighbours share a prefix.  Their next input token is the parent's until
        the caller writes another into `output_ids` (and into their own lists).  What the parent's launched steps gave has to
        have been read: the children take over its output as it is known.  None when request slots or cache do not suffice."""
        parent = self.reqs[index]
        if parent.finished():
            raise RuntimeError(f"fork: request {parent.rid} has finished")
        if parent.launched_tokens > len(parent.output_ids):
            raise RuntimeError(f"fork: request {parent.rid} has launched steps whose results are unread; drain them first")
        slots = fork_request(self.token_to_kv_pool_allocator.get_kvcache(), self.req_to_token_pool,
                             self.token_to_kv_pool_allocator, parent.req_pool_idx, n)
        if slots is None:
            return None
        children = []
        for k, slot in enumerate(slots):
            req = copy.copy(parent)
            req.rid = f"{parent.rid}.{parent.num_forks + k + 1}"
            req.num_forks = 0
            req.req_pool_idx = slot
            for name in ("origin_input_ids", "output_ids", "fill_ids", "prefix_indices", "token_times", "prior_output_ids",
                         "prior_token_times"):
                setattr(req, name, list(getattr(parent, name)))
            children.append(req)
        parent.num_forks += len(children)
        rows = list(range(index + 1)) + [index] * n + list(range(index + 1, len(self.reqs)))
        self.reqs = self.reqs[:index + 1] + children + self.reqs[index + 1:]
        self.seq_lens_host = [self.seq_lens_host[i] for i in rows]
        self.seq_lens_sum = sum(self.seq_lens_host)
        self.req_pool_indices = self._h2d([r.req_pool_idx for r in self.reqs], torch.int64)
        idx = self._h2d(rows, torch.int64)
        self.seq_lens = self.seq_lens[idx]
        if self.output_ids is not None:
            self.output_ids = self.output_ids[idx]
        return children

    def compact_req(self, index: int, keep: Sequence[int]) -> bool:
        """Request `index` of a decode batch goes on, between two steps, with its cached tokens at `keep` only (ascending indices
        into what is cached; memory_pool.compact_request).  Its next tokens stand at the positions that they would have had:
        the keys that are left are rotated for those.  A step with such a request runs without its CUDA graph.  False when the
        cache does not suffice."""
        req = self.reqs[index]
        if req.finished():
            raise RuntimeError(f"compact: request {req.rid} has finished")
        if not compact_request(self.token_to_kv_pool_allocator.get_kvcache(), self.req_to_token_pool,
                               self.token_to_kv_pool_allocator, req.req_pool_idx, keep):
            return False
        req.dropped_tokens += self.seq_lens_host[index] - len(keep)
        self.seq_lens_host[index] = len(keep)
        self.seq_lens_sum = sum(self.seq_lens_host)
        self.seq_lens = self._h2d(self.seq_lens_host, torch.int64)  # (a new one: a launched step may read the old)
        self._compacted = True
        return True

    def _position_offsets(self) -> Optional[torch.Tensor]:
        dropped = [r.dropped_tokens for r in self.reqs] if self._compacted else []
        self._compacted = any(dropped)
        return self._h2d(dropped, torch.int64) if self._compacted else None

    def _shared_prefix(self) -> Optional[SharedPrefix]:
        groups = self.token_to_kv_pool_allocator.shared_prefix([r.req_pool_idx for r in self.reqs])
        if groups is None:
            return None
        if self._shared is None or self._shared[0] != groups:  # lists of a few steps are the same
            indptr, lens = _joined_alone(*groups)
            self._shared = (groups, SharedPrefix(self._h2d(indptr, torch.int32), self._h2d(lens, torch.int64), max(lens)), indptr, lens)
        _, shared, indptr, lens = self._shared
        return dataclasses.replace(shared, tokens=ops.attn_shared_tokens(indptr, lens, self.seq_lens_host))

    def filter_batch(self, keep_indices: Optional[List[int]] = None):
        if keep_indices is None:
            keep_indices = [i for i, r in enumerate(self.reqs) if not r.finished()]
        if len(keep_indices) == len(self.reqs):
            return
        if not keep_indices:
            self.reqs = []
            self.req_pool_indices = self.seq_lens = self.output_ids = None
            self.seq_lens_sum = 0
            self.seq_lens_host = []
            return
        self.reqs = [self.reqs[i] for i in keep_indices]
        self.seq_lens_host = [self.seq_lens_host[i] for i in keep_indices]
        idx = self._h2d(keep_indices, torch.int64)
        self.req_pool_indices = self.req_pool_indices[idx]
        self.seq_lens = self.seq_lens[idx]
        if self.output_ids is not None:
            self.output_ids = self.output_ids[idx]
        self.seq_lens_sum = sum(self.seq_lens_host)

    def merge_batch(self, other: "ScheduleBatch"):
        self._compacted |= other._compacted
        if self.is_empty():
            self.reqs = list(other.reqs)
            self.req_pool_indices, self.seq_lens = other.req_pool_indices, other.seq_lens
            self.output_ids = other.output_ids
            self.seq_lens_sum = other.seq_lens_sum
            self.seq_lens_host = list(other.seq_lens_host)
            return
        self.req_pool_indices = torch.cat([self.req_pool_indices, other.req_pool_indices])
        self.seq_lens = torch.cat([self.seq_lens, other.seq_lens])
        if self.output_ids is not None and other.output_ids is not None:
            self.output_ids = torch.cat([self.output_ids, other.output_ids])
        self.seq_lens_sum += other.seq_lens_sum
        self.seq_lens_host = self.seq_lens_host + list(other.seq_lens_host)
        self.reqs.extend(other.reqs)

    def get_model_worker_batch(self) -> ModelWorkerBatch:
        global _bid
        _bid += 1
        extend = self.forward_mode.is_extend()
        return ModelWorkerBatch(
            bid=_bid, forward_mode=self.forward_mode, input_ids=self.input_ids,
            req_pool_indices=self.req_pool_indices, seq_lens=self.seq_lens,
            out_cache_loc=self.out_cache_loc, seq_lens_sum=self.seq_lens_sum,
            shared_prefix=None if extend else self._shared_prefix(),
            position_offsets=None if extend else self._position_offsets(),
            extend_num_tokens=self.extend_num_tokens if extend else None,
            extend_seq_lens=self.extend_lens if extend else None,
            extend_prefix_lens=self.prefix_lens if extend else None,
            extend_logprob_start_lens=[0] * len(self.reqs) if extend else None,
            gather_logits=getattr(self, "gather_logits", True),
            extend_logit_rows=getattr(self, "extend_logit_rows", None) if extend else None)


def _joined_alone(indptr, lens):
    """Group lists without requests that share nothing at both ends, those between two groups as one: a plan holds so many."""
    out, sizes = [], []
    for start, n in zip(indptr, lens):
        if n or (sizes and sizes[-1]):
            out.append(start)
            sizes.append(n)
    end = indptr[-1]
    if sizes and not sizes[-1]:
        end = out.pop()
        sizes.pop()
    return out + [end], sizes


def _cumsum(xs):
    s = 0
    for x in xs:
        s += x
        yield s
