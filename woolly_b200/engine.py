"""Continuous-batching generation on top of the multi-session runtime.

The reference serves one request at a time: `InferenceSession::infer_batch`
(woolly-core/src/session.rs:260-277) loops over its sequences and the server's
decode loop (woolly-server/src/handlers/inference.rs:371-438) calls
`InferenceEngine::infer` once per generated token, re-reading one shared KV
cache.  Here every request owns a session (its own paged KV cache on the
GPU); `BatchEngine.step()` admits waiting requests, prefills them, and then
runs ONE batched decode forward over every running request, so requests join
and leave the batch between steps (continuous batching).

Sampling follows the server's `sample_next_token` (inference.rs:441-483) and
its helpers (softmax_with_temperature, apply_top_k_filtering,
apply_top_p_filtering: inference.rs:551-630): temperature floor 0.01, top-k
by the k-th largest probability, top-p by the first prefix whose cumulative
probability exceeds p, greedy (temperature == 0) as the last index of the
largest probability, and a stop on token ids below 3 (inference.rs:414-418).
Where they leave nothing to choose from, the reference takes the last index;
here it is the last whose logit is not -inf, so that a closed token is never
picked.

Before sampling, a request's logits may go through rules that the reference
does not have: penalties for tokens that its prompt or output holds, biases and
a grammar's mask of the tokens that may follow (GenerationConfig; apply_rules on
the host, wl_process_logits on the GPU).
"""
from __future__ import annotations

from dataclasses import dataclass, field

import numpy as np

from ._lib import WL_ERR_OUT_OF_MEMORY, WoollyError


@dataclass
class GenerationConfig:
    """The server's generation knobs (inference.rs:25-27, 180-182)."""
    max_tokens: int = 16
    temperature: float = 0.0   # 0: greedy
    top_k: int = 0             # 0: off
    top_p: float = 1.0         # 1: off
    eos_below: int = 3         # stop once a token id < eos_below is produced (0: never)
    seed: int = 0              # per-request sampling stream
    repetition_penalty: float = 1.0  # logits of seen tokens: divided if positive, else multiplied (1: off)
    presence_penalty: float = 0.0    # taken off the logits of produced tokens, once
    frequency_penalty: float = 0.0   # and once for each time that they were produced
    logit_bias: dict | None = None   # token id -> added to its logit; below -1e38 (-inf) the token is closed
    # callable(tokens produced so far) -> ids that may follow, a boolean mask over the
    # vocabulary, or None for any; an empty answer ends the request ("constraint")
    allowed: object = None

    def has_rules(self) -> bool:
        return (self.repetition_penalty != 1.0 or self.presence_penalty != 0.0
                or self.frequency_penalty != 0.0 or bool(self.logit_bias) or self.allowed is not None)


def softmax_with_temperature(logits: np.ndarray, temperature: float) -> np.ndarray:
    """inference.rs:551-565 (f32, max-subtracted)."""
    t = np.float32(max(temperature, 0.01))
    x = np.asarray(logits, np.float32)
    e = np.exp((x - x.max()) / t).astype(np.float32)
    return (e / e.sum(dtype=np.float32)).astype(np.float32)


def apply_top_k(probs: np.ndarray, k: int) -> np.ndarray:
    """inference.rs:568-591: zero probabilities below the k-th largest, renormalise."""
    if k == 0 or k >= probs.size:
        return probs
    thr = np.sort(probs)[::-1][k - 1]
    p = np.where(probs < thr, np.float32(0), probs).astype(np.float32)
    s = p.sum(dtype=np.float32)
    return (p / s).astype(np.float32) if s > 0 else p


def apply_top_p(probs: np.ndarray, top_p: float) -> np.ndarray:
    """inference.rs:594-630: keep the shortest prefix (by descending
    probability) whose cumulative sum exceeds p; when no prefix exceeds p the
    reference keeps nothing (all zeros), and so does this."""
    if top_p >= 1.0:
        return probs
    order = np.argsort(-probs, kind="stable")
    cum = np.float32(0)
    cut = 0
    for i, idx in enumerate(order):
        cum = np.float32(cum + probs[idx])
        if cum > top_p:
            cut = i + 1
            break
    p = np.zeros_like(probs)
    keep = order[:cut]
    p[keep] = probs[keep]
    s = p.sum(dtype=np.float32)
    return (p / s).astype(np.float32) if s > 0 else p


def sample_next_token(logits: np.ndarray, cfg: GenerationConfig, rng: np.random.Generator) -> int:
    """sample_next_token (inference.rs:441-483) on one row of logits."""
    probs = softmax_with_temperature(logits, cfg.temperature)
    if cfg.top_k > 0:
        probs = apply_top_k(probs, cfg.top_k)
    if cfg.top_p < 1.0:
        probs = apply_top_p(probs, cfg.top_p)
    if cfg.temperature == 0.0:
        m = probs.max()
        # Rust max_by keeps the last maximum; zero (top-p kept nothing) and NaN are none
        return int(np.flatnonzero(probs == m)[-1]) if m > 0 else last_open(logits)
    return sample_from_distribution(probs, rng, logits)


def last_open(logits: np.ndarray) -> int:
    """The last index whose logit is not -inf (of a row without one, the last)."""
    i = np.flatnonzero(np.asarray(logits) != -np.inf)
    return int(i[-1]) if i.size else len(logits) - 1


def sample_from_distribution(probs: np.ndarray, rng: np.random.Generator,
                             logits: np.ndarray | None = None) -> int:
    """inference.rs:638-654: first index whose f32 running sum exceeds a
    uniform draw in [0, 1); the last index when none does (e.g. all zeros), of
    those that `logits` leaves open."""
    u = np.float32(rng.random(dtype=np.float32))
    cum = np.cumsum(probs, dtype=np.float32)
    hit = np.flatnonzero(cum > u)
    return int(hit[0]) if hit.size else last_open(probs if logits is None else logits)


RULE_MAX = 1e30     # penalties and biases of at most this leave logits finite in f32
BIAS_CLOSED = -1e38  # biases below this close their token


def open_mask(cfg: GenerationConfig, tokens, vocab: int) -> np.ndarray | None:
    """allowed_mask without the tokens that a bias closes."""
    m = allowed_mask(cfg, tokens, vocab)
    closed = [t for t, b in (cfg.logit_bias or {}).items() if b < BIAS_CLOSED]
    if closed:
        m = np.ones(vocab, bool) if m is None else m.copy()
        m[closed] = False
    return m


def allowed_mask(cfg: GenerationConfig, tokens, vocab: int) -> np.ndarray | None:
    """Boolean mask of the ids that may follow `tokens`, or None when any may."""
    if cfg.allowed is None:
        return None
    ids = cfg.allowed(list(tokens))
    if ids is None:
        return None
    ids = np.asarray(ids if isinstance(ids, np.ndarray) else list(ids))
    if ids.dtype == np.bool_:
        if ids.shape != (vocab,):
            raise ValueError(f"allowed() must give {vocab} truth values, got {ids.shape}")
        return ids
    m = np.zeros(vocab, bool)
    if ids.size:
        if ids.min() < 0 or ids.max() >= vocab:
            raise ValueError("allowed() gave an id outside the vocabulary")
        m[ids.astype(np.int64)] = True
    return m


def apply_rules(logits: np.ndarray, cfg: GenerationConfig, prompt, tokens,
                mask: np.ndarray | None = None) -> np.ndarray:
    """wl_process_logits' rules on one row, in f32: penalties for the tokens of
    the prompt (repetition) and of the output, biases, then the mask."""
    x = np.array(logits, np.float32, copy=True)
    V = x.size
    made = np.bincount(np.asarray([t for t in tokens if 0 <= t < V], np.int64), minlength=V)
    seen = made > 0
    seen[np.asarray([t for t in prompt if 0 <= t < V], np.int64)] = True
    r = np.float32(cfg.repetition_penalty)
    x[seen] = np.where(x[seen] > 0, x[seen] / r, x[seen] * r)
    hit = made > 0
    x[hit] -= np.float32(cfg.frequency_penalty) * made[hit].astype(np.float32) + np.float32(cfg.presence_penalty)
    with np.errstate(over="ignore"):  # a bias below f32's range is -inf
        for t, b in (cfg.logit_bias or {}).items():
            x[t] += np.float32(b)
    if mask is not None:
        x[~mask] = -np.inf
    return x


def pack_rules(requests, masks, vocab: int) -> dict:
    """The rules of a batch's rows (requests with cfg, prompt and tokens; their
    masks or None) as host arrays, keyed as process_logits and logit_params
    take them."""
    def starts(lists):
        return np.concatenate([[0], np.cumsum([len(x) for x in lists])]).astype(np.int32)

    def flat(lists, dtype):
        return np.concatenate([np.asarray(x, dtype) for x in lists]) if lists else np.zeros(0, dtype)
    hist = [r.prompt + r.tokens for r in requests]
    bias = [list((r.cfg.logit_bias or {}).items()) for r in requests]
    row, words = np.full(len(requests), -1, np.int32), []
    for i, m in enumerate(masks):
        if m is not None:
            row[i] = len(words)
            bits = np.zeros(-(-vocab // 32) * 32, np.uint8)
            bits[:vocab] = m
            words.append(np.packbits(bits, bitorder="little").view(np.uint32).view(np.int32))
    out = dict(
        params=dict(repetition=[r.cfg.repetition_penalty for r in requests],
                    presence=[r.cfg.presence_penalty for r in requests],
                    frequency=[r.cfg.frequency_penalty for r in requests], allowed_row=row),
        history=flat(hist, np.int32), history_start=starts(hist),
        prompt_lens=np.asarray([len(r.prompt) for r in requests], np.int32))
    if any(bias):
        with np.errstate(over="ignore"):
            out.update(bias_start=starts(bias), bias_tokens=flat([[t for t, _ in b] for b in bias], np.int32),
                       bias_values=flat([[v for _, v in b] for b in bias], np.float32))
    if words:
        out["allowed"] = np.stack(words)
    return out


@dataclass
class Request:
    rid: int
    prompt: list
    cfg: GenerationConfig
    rng: np.random.Generator
    tokens: list = field(default_factory=list)
    logits: list = field(default_factory=list)
    session: object = None
    done: bool = False
    reason: str = ""
    on_token: object = None  # callable(rid, token, done, reason) per produced token


class BatchEngine:
    """Continuous batching over a CudaTransformer (or any object with the same
    `forward_sessions` / `vocab_size` / `max_batch` interface).

    submit() queues a request; step() admits queued requests while sessions
    and batch room allow (each prefilled on its own, which yields its first
    token), then decodes one token for every other running request in one
    batched forward; run() steps until every request has finished.  A request
    finishes after cfg.max_tokens tokens, on a token id below cfg.eos_below,
    when its session's context is full, or when its grammar and its biases leave no
    token open ("constraint").  Its session is released at once, so a waiting
    request can take the slot on the next step.
    """

    def __init__(self, model, max_batch: int | None = None, session_factory=None,
                 max_context: int | None = None, keep_logits: bool = False,
                 device_sampling: bool = False):
        self.model = model
        self.max_batch = max_batch or model.max_batch
        if session_factory is None:
            from .model import Session
            session_factory = lambda: Session(model)  # noqa: E731
        self.new_session = session_factory
        self.max_context = max_context or getattr(model, "max_context", None)
        self.keep_logits = keep_logits
        # decode steps sample on the GPU (CudaTransformer.decode_sample): only
        # token ids cross to the host; the uniform draws still come from each
        # request's own stream, in the same order as host sampling
        self.device_sampling = device_sampling and not keep_logits and hasattr(model, "decode_sample")
        self.waiting: list[Request] = []
        self.running: list[Request] = []
        self.finished: dict[int, Request] = {}
        self._next = 0

    def submit(self, prompt, cfg: GenerationConfig | None = None, on_token=None) -> int:
        """Queues a request; `on_token(rid, token, done, reason)`, if given, is
        called as each of its tokens is produced (the server's streaming
        responses, inference.rs:271-357, forward tokens this way)."""
        prompt = [int(t) for t in prompt]
        if not prompt:
            raise ValueError("empty prompt (the reference's EMPTY_INPUT)")
        cfg = cfg or GenerationConfig()
        if not (1 / RULE_MAX <= cfg.repetition_penalty <= RULE_MAX):
            raise ValueError(f"repetition_penalty must lie in [{1 / RULE_MAX}, {RULE_MAX}]")
        if not (abs(cfg.presence_penalty) <= RULE_MAX and abs(cfg.frequency_penalty) <= RULE_MAX):
            raise ValueError(f"presence_penalty and frequency_penalty must lie within +-{RULE_MAX}")
        for t, b in (cfg.logit_bias or {}).items():
            if not (0 <= t < self.model.vocab_size()) or not b <= RULE_MAX:
                raise ValueError(f"logit_bias: token {t} outside the vocabulary, or its bias not up to {RULE_MAX}")
        r = Request(self._next, prompt, cfg, np.random.default_rng(cfg.seed), on_token=on_token)
        self._next += 1
        self.waiting.append(r)
        return r.rid

    # ---------------------------------------------------------------- internals
    def _mask(self, r: Request) -> np.ndarray | None:
        """The request's mask; one that leaves nothing ends the request."""
        m = open_mask(r.cfg, r.tokens, self.model.vocab_size())
        if m is not None and not m.any():
            r.done, r.reason = True, "constraint"
        return m

    def _emit(self, r: Request, row: np.ndarray, mask: np.ndarray | None) -> None:
        ruled = apply_rules(row, r.cfg, r.prompt, r.tokens, mask) if r.cfg.has_rules() else row
        tok = sample_next_token(ruled, r.cfg, r.rng)
        if self.keep_logits:
            r.logits.append(np.array(row, np.float32, copy=True))
        self._emit_token(r, tok)

    def _emit_token(self, r: Request, tok: int) -> None:
        r.tokens.append(int(tok))
        if len(r.tokens) >= r.cfg.max_tokens:
            r.done, r.reason = True, "length"
        elif r.cfg.eos_below and tok < r.cfg.eos_below:
            r.done, r.reason = True, "eos"
        elif self.max_context is not None and len(r.session) + 1 > self.max_context:
            r.done, r.reason = True, "context"
        if r.on_token is not None:
            r.on_token(r.rid, int(tok), r.done, r.reason)

    def _retire(self) -> None:
        keep = []
        for r in self.running:
            if r.done:
                r.session.close()
                r.session = None
                self.finished[r.rid] = r
            else:
                keep.append(r)
        self.running = keep

    def _admit(self) -> None:
        """Moves waiting requests to `running`, whose sessions the engine closes."""
        while self.waiting and len(self.running) < self.max_batch:
            r = self.waiting[0]
            if self.max_context is not None and len(r.prompt) >= self.max_context:
                self.waiting.pop(0)
                r.done, r.reason = True, "context"
                self.finished[r.rid] = r
                continue
            try:
                r.session = self.new_session()
            except WoollyError as e:
                if e.code == WL_ERR_OUT_OF_MEMORY:  # every session slot is taken
                    break
                raise
            self.waiting.pop(0)
            self.running.append(r)

    # ---------------------------------------------------------------- public
    def step(self) -> int:
        """One scheduler iteration; returns the number of tokens produced.

        An exception from a request's own part is raised once the others have
        finished the step (the first, of several).  One from its grammar or its
        prefill ends the request with the reason "error"; after one from on_token
        it goes on, its token being produced."""
        produced, errors = 0, []

        def alone(r, part, *args):
            n = len(r.tokens)
            try:
                return part(r, *args)
            except Exception as e:
                if len(r.tokens) == n:
                    r.done, r.reason = True, "error"
                errors.append(e)

        decoding = [r for r in self.running if r.tokens]
        try:
            self._admit()
            for r in self.running:  # prefill: the prompt's last row gives the first token
                if not r.tokens:
                    alone(r, self._prefill)
                    produced += len(r.tokens)
            # before anything is decoded, since a grammar may end its request or raise
            masks = {r.rid: alone(r, self._mask) for r in decoding}
            decoding = [r for r in decoding if not r.done]
            if decoding and self.device_sampling:
                kw = {}
                if any(r.cfg.has_rules() for r in decoding):
                    kw["rules"] = pack_rules(decoding, [masks[r.rid] for r in decoding], self.model.vocab_size())
                cf = [r.cfg for r in decoding]
                u = [np.float32(r.rng.random(dtype=np.float32)) if r.cfg.temperature != 0.0 else 0.0
                     for r in decoding]
                toks = self.model.decode_sample([r.session for r in decoding],
                                                [r.tokens[-1] for r in decoding],
                                                [c.temperature for c in cf], [c.top_k for c in cf],
                                                [c.top_p for c in cf], u, **kw)
                for r, tok in zip(decoding, toks):
                    alone(r, self._emit_token, tok)
                    produced += 1
            elif decoding:
                outs = self.model.forward_sessions([r.session for r in decoding],
                                                   [[r.tokens[-1]] for r in decoding])
                for r, row in zip(decoding, outs):
                    n = len(r.tokens)
                    alone(r, self._emit, np.asarray(row).reshape(-1), masks[r.rid])
                    produced += len(r.tokens) - n
        finally:
            self._retire()
        if errors:
            raise errors[0]
        return produced

    def _prefill(self, r: Request) -> None:
        mask = self._mask(r)
        if not r.done:
            row = self.model.forward_sessions([r.session], [r.prompt])[0]
            self._emit(r, np.asarray(row).reshape(-1)[-self.model.vocab_size():], mask)

    def idle(self) -> bool:
        return not self.waiting and not self.running

    def run(self, max_steps: int = 1_000_000) -> dict[int, list]:
        for _ in range(max_steps):
            if self.idle():
                break
            self.step()
        return {rid: r.tokens for rid, r in sorted(self.finished.items())}

    def stream(self, prompt, cfg: GenerationConfig | None = None):
        """Submits a request and yields its tokens as they are produced,
        stepping the whole engine (other requests advance in the same batched
        steps)."""
        got: list = []
        rid = self.submit(prompt, cfg, on_token=lambda _r, tok, _d, _why: got.append(tok))
        while rid not in self.finished:
            self.step()
            while got:
                yield got.pop(0)
        while got:
            yield got.pop(0)

    def close(self) -> None:
        for r in self.running:
            if r.session is not None:
                r.session.close()
                r.session = None
        self.running = []
