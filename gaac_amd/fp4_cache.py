"""Slot cache of one attention layer in 4 bits, with the methods of CompressedKVCache (kv_cache.py): 3.76 times smaller than bf16 where that one is lossless
and 1.4 times smaller.

32 consecutive channels of a token and head share a power of two 2^E, the smallest with max |x| < 7 * 2^E, from -125 to 125; an element is held as its sign and the
nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^E, ties to the even code (OCP MXFP4, 4.25 bits an element).  A block with a NaN or an infinity reads as NaN.  A
token is quantised as it is written and by itself: what the cache holds of it does not depend on whether it came in a prompt or as a decode step's token.  The
values are numbers of bf16, so reading them back rounds nothing.

Slot s owns cache heads [s*n_kv, (s+1)*n_kv); a head is a row of tiles of 32 tokens, K and V of a tile in 4352 bytes next to each other (csrc/fp4.hip).
append and attention take the batch's slot map and the slots' lengths from device memory and never return to the host, so a decode step can be captured in a
HIP graph.  Calls on one cache must be ordered on one stream where one of them writes; attention may run on several streams at
once, and in several graphs: its scratch is the call's own, and the counters by which the splits of a row find the last of them are one set for each stream and one
for each captured call.  A call that is not captured makes its stream's set, and sees to it that READY sets lie ready for captured calls of as many rows; a captured call that finds
none, or after CAPTURES of them, takes a launch more instead; captured_counters and give_back return the sets of graphs that are dropped.  128 bytes a row and kv head of a call, beside its partials: scratch of the calls, not of the slots.
No call has a backward pass: tensors whose gradient it would lose, in either mode of differentiation, are refused."""
from __future__ import annotations
import contextlib
import functools
import threading
import torch
from . import _lib
from .codec import D
from .kernel import GMAX

T = 32                          # tokens per tile
ROW_BYTES = D // 2 + D // 32    # bytes of a token and head of K or of V: codes and exponents
TILE_BYTES = 2 * T * ROW_BYTES
LINE = 32                       # words from one counter of attention to the next
CAPTURES = 64                   # captured calls of attention that get counters of their own
READY = 16                      # sets of counters that calls outside of captures keep ready for calls inside, which cannot make any

_LOCK = threading.Lock()        # over the sets that lie ready


@functools.lru_cache(maxsize=None)
def _side_stream(device: torch.device) -> torch.cuda.Stream:
    return torch.cuda.Stream(device)      # (one for all caches: the allocator keeps memory apart by streams)


@functools.lru_cache(maxsize=1024)
def choose_nsplit(B: int, n_kv: int, S: int, G: int = 4) -> int:
    """Splits for each of B rows, S tokens in the longest, G query heads a kv head, which the launch then shares out by length (csrc/fp4.hip).  Measured, 8 kv heads and G 4 unless noted, us:
      * up to 1500 tokens none (1000 tokens: 7.0, against 7.8 with 7 splits; 8 rows of 1500: 8.8, with 4 9.5; but 1 row of 1500 alone 8.5, with 11 8.1);
      * heads that fill half of the chip by themselves: none, since a split's start and merge cost more than even shares save (32 rows of 300..6000: 23.7, against
        26.2 with 2; 24 of 2000..16000: 52.4 and 53.4; 64 of 2000..16000: 106 and 115), but not where a single row may take as long as all (from 32768 tokens);
      * otherwise one block per CU (8 rows of 7000..8192: 17.8 with 4, 22.9 with 2, 18.0 with 8), two for long rows, whose tiles are worth more loads in flight (16 rows of 4096..65536: 101
        with 4, 111 with 2; 8 of 32768: 50.8 with 8, 50.2 with 4);
      * but of few heads no more splits than their merge by one block is worth: 16 (4096 tokens: 8.2, with 32 8.7; 16384: 10.7 and 10.1), from 24576 tokens 32 (65536: 18.2, with 16 21.8; 32768 x
        1: 11.0, with 16 13.2, with 256 24; G 16 18.4, 19.1 and 73), and for G up to 4 64 from 65536 (131072 x 1: 16.1, with 32 19.8), 128 from 262144 (20.8, with 64 22.1; 10^6 x 1: 37.2,
        with 64 57, with 256 40), for more heads to merge from four times these lengths (G 16, 131072 x 1: 27, with 64 29; 262144: 35, with 32 39; 10^6: 70, with 128 62)."""
    H = B * n_kv
    if S <= 1500: return 1
    if H > 128: return 1 if S < 32768 else 2
    s = S if G <= 4 else S // 4
    few = 16 if S < 24576 else 32 if s < 65536 else 64 if s < 262144 else 128 if s < 1 << 21 else 256
    return max(1, min((512 if H * S >= 1 << 22 else 256) // H, S // 128, few))


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [., heads, 128] as the kernels read it: channels next to each other, heads and tokens any multiple of 16 bytes apart; other layouts are copied."""
    (rs, hs, one), shape = x.stride(), x.shape
    if one == 1 and (shape[1] == 1 or hs % 8 == 0) and (shape[0] == 1 or rs % 8 == 0) and x.data_ptr() % 16 == 0: return x
    return x.clone(memory_format=torch.contiguous_format)


def _strides(x: torch.Tensor) -> tuple[int, int]:
    """(head stride, row stride)."""
    return x.stride(1) if x.shape[1] > 1 else 0, x.stride(0) if x.shape[0] > 1 else 0


class FP4KVCache:
    def __init__(self, n_slots: int, n_kv: int, capacity: int, device="cuda"):
        """n_slots sequences of up to `capacity` tokens (rounded up to whole tiles), n_kv cache heads each."""
        _lib.load()      # fail here, not at the first decode step, if the native library is missing
        if n_slots < 1 or n_kv < 1 or capacity < 1: raise RuntimeError(f"FP4KVCache expects slots, kv heads and capacity of at least 1, got {n_slots}, {n_kv}, {capacity}")
        self.n_slots, self.n_kv = n_slots, n_kv
        self.tiles = -(-capacity // T)
        self.cap = self.tiles * T
        self.H = n_slots * n_kv
        self.data = torch.zeros(self.H, self.tiles, TILE_BYTES, dtype=torch.uint8, device=device)
        self.lens = torch.zeros(n_slots, dtype=torch.int32, device=device)          # tokens per slot; the caller may set them: below 0 counts as 0, above cap as cap
        # set by append instead of writing: bit 0 = a slot was full or its length below 0, bit 1 = a slot twice in a batch, bit 2 = no such slot
        self.overflow = torch.zeros(1, dtype=torch.int32, device=device)
        self._no_counters()

    def _no_counters(self):
        self._tickets = {}                                           # stream -> counters, zero between launches
        self._ready, self._ready_words, self._given = [], 0, []      # the same for captured calls: sets that lie ready and their size, sets that a captured call has
        self._noted = {}                                             # thread -> the sets that calls inside its captured_counters() have taken

    def __getstate__(self):      # counters belong to streams and graphs of this process
        return {k: v for k, v in self.__dict__.items() if k not in ("_tickets", "_ready", "_ready_words", "_given", "_noted")}

    def __setstate__(self, state):
        self.__dict__.update({k: v for k, v in state.items() if k not in ("_tickets", "_spare", "_captured")})      # (what caches saved earlier hold)
        self._no_counters()

    @property
    def _captured(self) -> int:
        return len(self._given)

    def _counters(self, n: int) -> torch.Tensor | None:
        """Counters of an attention launch, n of them: launches on one stream are in order and share theirs; a captured call may be replayed beside any other."""
        words = n * LINE
        if torch._C._cuda_isCurrentStreamCapturing():
            with _LOCK:
                if not self._ready or words > self._ready_words: return None
                have = self._ready.pop()
                self._given.append(have)
                noted = self._noted.get(threading.get_ident())
                if noted is not None: noted.append(have)
                return have
        stream = _lib.stream()
        have = self._tickets.get(stream)
        if have is None or have.numel() < words: have = self._tickets[stream] = torch.zeros(words, dtype=torch.int32, device=self.data.device)
        if words > self._ready_words or len(self._ready) < READY: self._make_ready(words)
        return have

    @contextlib.contextmanager
    def captured_counters(self):
        """The sets of counters that attention() takes inside, in a list: for a capture whose graph will be dropped, and give_back then."""
        me = threading.get_ident()
        if me in self._noted: raise RuntimeError("captured_counters within captured_counters")
        self._noted[me] = taken = []
        try: yield taken
        finally: del self._noted[me]

    def give_back(self, counters: list):
        """Counters of captured calls whose graph has run for the last time, the GPU being done with it: later captures take them again."""
        with _LOCK:
            for c in counters:
                at = next((i for i, s in enumerate(self._given) if s is c), None)
                if at is None: raise RuntimeError("give_back expects counters that captured calls of this cache hold")
                self._given.pop(at)
                if c.numel() >= self._ready_words: self._ready.append(c)      # (smaller ones are no longer handed out)

    def _unused(self, counters: torch.Tensor | None):
        """Counters of a captured call that was not made after all."""
        with _LOCK: held = any(s is counters for s in self._given)
        if not held: return
        self.give_back([counters])
        noted = self._noted.get(threading.get_ident(), [])
        noted[:] = [s for s in noted if s is not counters]

    def _make_ready(self, words: int):
        with _LOCK:
            if words > self._ready_words: self._ready, self._ready_words = [], words
            missing = min(READY, CAPTURES - len(self._given)) - len(self._ready)
            if missing < 1: return
            side = _side_stream(self.data.device)      # zero before this call returns, whatever the current stream still has to do: a graph may run on any
            with torch.cuda.stream(side): made = torch.zeros(missing, self._ready_words, dtype=torch.int32, device=self.data.device)
            side.synchronize()
            self._ready.extend(made.unbind(0))

    @staticmethod
    def bytes_per_slot(n_kv: int, capacity: int) -> int:
        """Device bytes one slot occupies: its tiles and its length, which is all that a cache holds for its slots."""
        return n_kv * -(-capacity // T) * TILE_BYTES + 4

    def _check(self, what: str, k: torch.Tensor, v: torch.Tensor):
        if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or k.shape != v.shape or k.dim() != 3 or tuple(k.shape[1:]) != (self.n_kv, D):
            raise RuntimeError(f"{what} expects k, v bf16 [., {self.n_kv}, {D}], got {k.dtype} {list(k.shape)} and {v.dtype} {list(v.shape)}")

    # ------------------------------------------------------------------ prefill
    def prefill(self, slot: int, k: torch.Tensor, v: torch.Tensor):
        """Put a whole prompt into `slot`, replacing what the slot held: k, v bf16 [L, n_kv, D] in the model's token-major layout, through any strides of whole
        16 bytes.  One launch, no wait."""
        if (_lib._calls or _lib.calls()).fp4_prefill(self, slot, k, v, _lib.stream): return
        self._check("prefill", k, v)
        L = k.shape[0]
        if not 0 <= slot < self.n_slots: raise RuntimeError(f"prefill expects a slot in 0..{self.n_slots - 1}, got {slot}")
        if L > self.cap: raise RuntimeError(f"prompt has {L} tokens, a slot holds {self.cap}")
        _lib.no_backward("prefill", k, v)
        with _lib.on_device(self.data, k, v):
            k, v = _rows(k), _rows(v)
            (k_hs, k_rs), (v_hs, v_rs) = _strides(k), _strides(v)
            _lib.call("gaac_fp4_store", k, v, k_hs, k_rs, v_hs, v_rs, L, self.n_kv, self.tiles, self.data[slot * self.n_kv], self.lens[slot:], _lib.stream)

    # ------------------------------------------------------------------ decode step
    def append(self, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
        """Decode-step write: batch row b adds the token k[b], v[b] (bf16 [B, n_kv, D], through any strides of whole 16 bytes) to slot slots[b] (int32 [B]; -1 leaves the
        row out).  One launch, no wait.  A row whose slot is full, stands earlier in the batch already or does not exist is left out, and check_capacity raises."""
        if (_lib._calls or _lib.calls()).fp4_append(self, slots, k, v, _lib.stream): return
        self._check("append", k, v)
        if slots.dtype != torch.int32 or slots.dim() != 1 or slots.shape[0] != k.shape[0]: raise RuntimeError("append expects slots int32 [B]")
        _lib.no_backward("append", k, v)
        if k.shape[0] == 0: return
        with _lib.on_device(self.data, slots, k, v):
            k, v = _rows(k), _rows(v)
            (k_hs, k_bs), (v_hs, v_bs) = _strides(k), _strides(v)
            _lib.call("gaac_fp4_append", slots.contiguous(), slots.shape[0], self.n_slots, self.n_kv, k, v, k_bs, k_hs, v_bs, v_hs, self.lens, self.tiles, self.cap,
                      self.data, self.overflow, _lib.stream)

    def attention(self, q: torch.Tensor, slots: torch.Tensor, scale: float, max_len: int | None = None, nsplit: int | None = None) -> torch.Tensor:
        """Decode-step read: bf16 [B, n_q, D] queries, row b over everything slot slots[b] holds; returns bf16 [B, n_q, D].  A row whose slot is -1 or empty is 0, one
        whose slot does not exist NaN.  max_len, the longest row if the caller knows it, only picks the split count when nsplit is not given."""
        shape = q.shape
        if nsplit is None: nsplit = choose_nsplit(shape[0] or 1, self.n_kv, min(int(max_len), self.cap) if max_len else self.cap, shape[1] // self.n_kv) if len(shape) == 3 else 1
        tickets = out = None
        if nsplit == 1: out = (_lib._calls or _lib.calls()).fp4_attend(self, q, slots, scale, 1, None, _lib.stream)
        elif nsplit > 1 and q.is_cuda and q.device == self.data.device and q.device.index == torch._C._cuda_getDevice():
            tickets = self._counters(shape[0] * self.n_kv if shape else 0)
            try: out = (_lib._calls or _lib.calls()).fp4_attend(self, q, slots, scale, nsplit, tickets, _lib.stream)
            except BaseException:
                self._unused(tickets)
                raise
        if out is not None: return out
        try: return self._attention(q, slots, scale, nsplit, tickets)
        except BaseException:
            self._unused(tickets)
            raise

    def _attention(self, q, slots, scale, nsplit, tickets) -> torch.Tensor:
        """attention, where the binding does not make the call.  tickets: the call's counters, if it has some already."""
        if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[2] != D: raise RuntimeError(f"attention expects q bf16 [B, n_q, {D}], got {q.dtype} {list(q.shape)}")
        B, n_q, _ = q.shape
        if n_q % self.n_kv or not 1 <= n_q // self.n_kv <= GMAX: raise RuntimeError(f"GQA group size must be 1..{GMAX}")
        if slots.dtype != torch.int32 or slots.dim() != 1 or slots.shape[0] != B: raise RuntimeError("attention expects slots int32 [B]")
        _lib.no_backward("attention", q)
        if nsplit < 1: raise RuntimeError(f"attention expects at least one split, got {nsplit}")
        with _lib.on_device(self.data, q, slots):
            out = torch.empty(B, n_q, D, dtype=q.dtype, device=q.device)
            if B == 0: return out
            partials = None
            if nsplit > 1:
                partials = torch.empty(B * nsplit * n_q * (D + 2), dtype=torch.float32, device=q.device)
                if tickets is None: tickets = self._counters(B * self.n_kv)
            q = q if q.is_contiguous() and q.data_ptr() % 16 == 0 else q.clone(memory_format=torch.contiguous_format)
            _lib.call("gaac_fp4_attn", self.data, self.lens, slots.contiguous(), self.n_slots, self.tiles, self.cap, q, B, n_q, self.n_kv, float(scale), int(nsplit), partials,
                      tickets, out, _lib.stream)
            return out

    # ------------------------------------------------------------------ housekeeping
    def check_capacity(self, used: int | None = None):
        """Raises if append had to leave a row out since the cache was made (waits for the stream).  used: the word, if the caller fetched it already."""
        hit = int(self.overflow) if used is None else used
        if hit:
            raise RuntimeError("4-bit KV cache lost data:" + (" a sequence grew past the slot's token capacity, or its length was set below 0;" if hit & 1 else "") +
                               (" a slot stood twice in a batch;" if hit & 2 else "") + (" a batch named a slot that does not exist" if hit & 4 else ""))

    def decompress(self, slot: int) -> tuple[torch.Tensor, torch.Tensor]:
        """The K and V that `slot` holds, bf16 [L, n_kv, D] each (waits for the stream, to read the slot's length)."""
        both = (_lib._calls or _lib.calls()).fp4_read(self, slot, _lib.stream)
        if both is not None: return both
        if not 0 <= slot < self.n_slots: raise RuntimeError(f"decompress expects a slot in 0..{self.n_slots - 1}, got {slot}")
        L = max(0, min(int(self.lens[slot]), self.cap))
        k = torch.empty(L, self.n_kv, D, dtype=torch.bfloat16, device=self.data.device)
        v = torch.empty_like(k)
        if L:
            with _lib.on_device(self.data):
                _lib.call("gaac_fp4_load", self.data[slot * self.n_kv], L, self.n_kv, self.tiles, k, v, D, self.n_kv * D, D, self.n_kv * D, _lib.stream)
        return k, v

    def stats(self) -> dict:
        """Occupancy (the keys of CompressedKVCache.stats): bytes_used counts codes and exponents of the tokens held."""
        tokens = int(self.lens.clamp(0, self.cap).sum())
        used, bf16 = tokens * self.n_kv * 2 * ROW_BYTES, tokens * self.n_kv * 2 * D * 2
        return dict(tokens=tokens, bytes_used=used, bf16_bytes=bf16, ratio=bf16 / max(1, used))
