"""A policy that acts on a stream of frames: every LLM layer keeps the keys and values of past frames in an 8-bit paged cache
(kernels.KV8Cache), positions have three axes (time, row, column), and a new frame's tokens attend to all that is remembered.

    python -m yanlongvla_b200.stream --robots 2 --frames 8 [--llm-layers 24] [--window 4] [--candidates 8]

runs the policy of `policy` (random weights, synthetic frames) with a memory and prints the time per frame; with a window it
remembers no more than that many frames, with candidates it forms several action chunks of each observation. The kernels:
rope_axes turns the queries, kv8_append turns and stores the keys and stores the values, kv8_attention reads the cache; of a memory
with a pool of pages kv8_fork shares, kv8_reserve and kv8_copy give pages, kv8_compact and kv8_free forget. All lengths and
positions live on the device, so a step can be captured in a CUDA graph: what a capture records moves them on at each
replay, and StreamMemory.reserve(), called before each replay (with what the step keeps of the past, where it forgets), keeps the
host's count and checks the capacity.
"""
import argparse
import operator

import torch

from . import kernels as K


class StreamMemory:
    """Caches of every LLM layer for `robots` sequences of up to `max_tokens` tokens. Without `pages`, pages are assigned once: block i
    of robot b is page b * blocks + i of each layer. With it, all robots share a pool of that many pages and get them as
    they remember more; such a memory can be forked and thinned out (fork, keep, keep_recent). Its operators are the kernels in
    every runtime of the policy, the one of PyTorch operations among them."""

    def __init__(self, c, robots, max_tokens, device='cuda', theta=10000.0, max_frames=4096, pages=None):
        D = c.llm_hidden // c.llm_heads
        self.c, self.robots, self.max_tokens, self.tokens = c, robots, max_tokens, 0
        blocks = -(-max_tokens // K.KV8_BLOCK)
        self.pages = None if pages is None else K.KV8Pages.empty(pages, device)
        self.caches = [K.KV8Cache.empty(robots * blocks if pages is None else pages, c.llm_kv_heads, D, device) for _ in range(c.llm_layers)]
        if pages is None:
            self.table = torch.arange(robots * blocks, dtype=torch.int32, device=device).view(robots, blocks)
        else:
            self.table = self.pages.table(robots, blocks)
        self.count = None                                                        # tokens of the current frame, where not all of it
        self.served = torch.ones(robots, dtype=torch.bool, device=device)        # which robots the pool had pages for in the current frame
        # a quarter of the frequencies for time, the rest split between rows and columns
        time = D // 8
        row = (D // 2 - time + 1) // 2
        side = int(c.image_tokens ** 0.5)
        span = max(max_frames, c.cameras * side + c.lang_tokens)
        self.rope = K.RopeAxes(*K.RopeAxes.tables(span, D, theta, device), (time, row, D // 2 - time - row))
        self.max_frames, self.frames = min(max_frames, span), 0
        self.start = torch.zeros(robots, dtype=torch.int32, device=device)       # tokens remembered before the current frame
        self.lens = torch.zeros(robots, dtype=torch.int32, device=device)        # and with it
        # positions of a frame's tokens: image tokens by camera, row and column, then the instruction behind them on both axes
        i = torch.arange(c.image_tokens, dtype=torch.int32)
        rows = torch.cat([i // side] * c.cameras + [side + torch.arange(c.lang_tokens, dtype=torch.int32)])
        cols = torch.cat([i % side + side * k for k in range(c.cameras)] + [side * c.cameras + torch.arange(c.lang_tokens, dtype=torch.int32)])
        pos = torch.stack((torch.full_like(rows, -1), rows, cols)).to(device)          # begin_frame moves the time on
        self.pos = pos[:, None].expand(3, robots, pos.shape[1]).contiguous()

    def reserve(self, kept=None):
        """Count the next frame in on the host; refused where it does not fit. begin_frame calls it, except in a capture, which runs
        nothing: call it before each replay of a captured step. kept: that step first keeps at most so many tokens of each robot (keep,
        keep_recent; 0: none), which a capture does not count either; where the pool might not hold them next to the old ones (see keep), the
        count stays. Frames of which a count was remembered (begin_frame) are counted in full; where that is too much, the longest
        memory's length is read from the device, behind the work of the current stream."""
        n = self.pos.shape[2]
        if kept is not None:
            kept = operator.index(kept)
            if kept < 0:
                raise K.TcqError(f'StreamMemory: {kept} tokens cannot be kept')
            if kept:
                self._pooled('keep')

        def held():
            return min(self.tokens, kept) if kept is not None and self._holds(kept) else self.tokens
        if held() + n > self.max_tokens and not torch.cuda.is_current_stream_capturing():
            self.tokens = self._longest()                                        # frames with a count held less than was counted
        if held() + n > self.max_tokens or self.frames >= self.max_frames:
            raise K.TcqError(f'StreamMemory: a frame of {n} tokens does not fit behind {held()} of {self.max_tokens} tokens, {self.frames} frames')
        self.tokens = held() + n
        self.frames += 1

    def _holds(self, n):
        """Whether the pool surely holds n tokens of every robot next to all that they may remember."""
        blocks = lambda tokens: -(-tokens // K.KV8_BLOCK)
        return n < 1 or self.robots * (blocks(self.tokens) + blocks(min(n, self.tokens))) <= self.pages.pages

    def _longest(self):
        """The longest memory's tokens, read from the device, and those of frames that were counted and are not there yet."""
        longest, last = torch.stack((self.lens.max(), self.pos[0, 0, 0])).tolist()
        return min(self.tokens, longest + (self.frames - 1 - last) * self.pos.shape[2])

    def begin_frame(self, frame=None, count=None):
        """Make room for the next frame: its tokens follow those remembered. On the device but for the check of the capacity.
        frame: the (B, T, ...) tensor that the layers will get; one of another batch or length is refused before anything moves.
        count (robots,) int32: each robot's tokens of the frame (0 .. its length), the rest is padding (None: all). A robot that the
        pool of pages does not serve remembers nothing of the frame, and its tokens attend to nothing (served (robots,) bool says which
        robots were served, device_error reports flag 2)."""
        n = self.pos.shape[2]
        if frame is not None and tuple(frame.shape[:2]) != (self.robots, n):
            raise K.TcqError(f'StreamMemory: a frame of {self.robots} robots with {n} tokens each expected, got {tuple(frame.shape[:2])}')
        if count is not None:
            self._ints('count', count, (self.robots,))
        if not torch.cuda.is_current_stream_capturing():
            self.reserve()
        self.pos[0] += 1
        self.start.copy_(self.lens)
        self.count = None if count is None else count.clamp(0, n)
        if self.pages is not None:
            want = torch.full_like(self.lens, n) if count is None else self.count
            self.count, copies = K.kv8_reserve(self.pages, self.table, self.lens, want)
            torch.eq(self.count, want, out=self.served)
            K.kv8_copy(self.caches, copies)
        self.lens += n if self.count is None else self.count

    def attend(self, layer, q, k, v):
        """The attention of one layer over everything remembered and the current frame (causal): q (B, T, heads * D) is turned in
        place, k and v (B, T, kv_heads * D) go into the layer's cache."""
        cache = self.caches[layer]
        K.kv8_append(cache, k, v, self.table, self.start, count=self.count, rope=self.rope, pos=self.pos)
        K.rope_axes(q, self.pos, self.rope, out=q)
        return K.kv8_attention(q, cache, self.table, self.lens, count=self.count)

    def _ints(self, name, t, shape):
        if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != self.lens.device:
            raise K.TcqError(f'StreamMemory: {name} must be int32 {shape} on {self.lens.device}, got {t.dtype} {tuple(t.shape)} on {t.device}')

    def _pooled(self, what):
        if self.pages is None:
            raise K.TcqError(f'StreamMemory: {what} needs a pool of pages (pages=)')

    def fork(self, parent):
        """Robot b's memory becomes what robot parent[b]'s is (parent (robots,) int32; below 0: empty), without copying it: pages are shared
        until one of the robots goes on in a begun block. For several continuations of one past."""
        self._pooled('fork')
        K.kv8_fork(self.pages, self.table, self.lens, parent)

    def keep(self, index, kept=None):
        """Remember only the tokens index[b, j], j < kept[b] (index (robots, n) int32, kept (robots,) int32 or None: all n; at most as
        many as robot b remembers), packed into pages of the pool, which takes the old ones back; positions in time and space
        stay what they were. A robot whose tokens the pool's free pages do not hold next to the old ones keeps its memory, and so do all
        behind it (device_error reports flag 2). A pool of robots * (blocks of all that they remember + blocks of n) pages serves all;
        where it may be smaller, the call reads a length back to know whether it did (not in a capture)."""
        self._pooled('keep')
        n = index.shape[-1] if index.dim() else 0
        self._ints('index', index, (self.robots, max(n, 1)))
        if kept is not None:
            self._ints('kept', kept, (self.robots,))
        if n > self.table.shape[1] * K.KV8_BLOCK:
            raise K.TcqError(f'StreamMemory: {n} tokens do not fit {self.max_tokens}')
        most = self.lens.clamp(max=n)
        kept = most if kept is None else kept.clamp(min=0).minimum(most)
        self._pack(index.contiguous(), kept, kept)

    def _pack(self, index, kept, move):
        """move (robots,): kept, or 0 for robots whose memory may stay as it is."""
        n = index.shape[1]
        table = self.pages.table(*self.table.shape)
        granted, _ = K.kv8_reserve(self.pages, table, torch.zeros_like(self.lens), move)
        K.kv8_compact(self.caches, self.table, self.lens, index, table, kept=granted)
        stays = granted < kept
        K.kv8_free(self.pages, self.table, self.lens, torch.where(stays, self.lens, 0))
        self.table.copy_(torch.where(stays[:, None], self.table, table))
        self.lens.copy_(torch.where(stays, self.lens, granted))
        if not torch.cuda.is_current_stream_capturing():
            self.tokens = min(self.tokens, n) if self._holds(n) else self._longest()

    def keep_recent(self, tokens):
        """Remember only the newest `tokens` tokens of each robot (0: none). Positions go on as if the others were still there. Robots that
        remember no more stay as they are; of the others' pages holds what keep says."""
        self._pooled('keep_recent')
        if tokens < 1:
            K.kv8_free(self.pages, self.table, self.lens, torch.zeros_like(self.lens))
            if not torch.cuda.is_current_stream_capturing():
                self.tokens = 0
            return
        tokens = min(tokens, self.table.shape[1] * K.KV8_BLOCK)
        kept = self.lens.clamp(max=tokens)
        at = torch.arange(tokens, dtype=torch.int32, device=self.lens.device)
        index = (self.lens - kept)[:, None] + at.minimum((kept - 1).clamp(min=0)[:, None])
        self._pack(index, kept, torch.where(self.lens > tokens, kept, 0))

    def forget(self):
        """Remember nothing, time starts anew. (In a capture the host's counts stay: reserve(kept=0) before a replay, and max_frames counts
        the frames of all replays.)"""
        if not torch.cuda.is_current_stream_capturing():
            self.tokens = self.frames = 0
        if self.pages is not None:
            K.kv8_free(self.pages, self.table, self.lens, torch.zeros_like(self.lens))
        self.lens.zero_()
        self.start.zero_()
        self.served.fill_(True)
        self.pos[0].fill_(-1)

    @property
    def bytes(self):
        return sum(t.numel() * t.element_size() for c in self.caches for t in (c.k, c.v, c.k_scale, c.v_scale))


def main(argv=None):
    from . import policy as P
    ap = argparse.ArgumentParser(description='run the policy on a stream of synthetic frames with an 8-bit memory')
    ap.add_argument('--robots', type=int, default=1)
    ap.add_argument('--frames', type=int, default=16)
    ap.add_argument('--window', type=int, default=0, help='frames remembered (0: all)')
    ap.add_argument('--candidates', type=int, default=1, help='action chunks formed of each observation')
    ap.add_argument('--vit-layers', type=int, default=P.PolicyConfig.vit_layers)
    ap.add_argument('--llm-layers', type=int, default=P.PolicyConfig.llm_layers)
    ap.add_argument('--dit-layers', type=int, default=P.PolicyConfig.dit_layers)
    a = ap.parse_args(argv)
    c = P.PolicyConfig(vit_layers=a.vit_layers, llm_layers=a.llm_layers, dit_layers=a.dit_layers)
    model, _, _ = P.build_policy(runtime='resident', c=c)
    n, window = c.prefix_tokens, a.window if 0 < a.window < a.frames else 0
    most = max(a.frames, 4096)                                                   # frames that positions are there for
    if window:
        # full and next to it what is kept of it
        blocks = -(-window * n // K.KV8_BLOCK) + -(-(window - 1) * n // K.KV8_BLOCK)
        memory = StreamMemory(c, a.robots, window * n, max_frames=most, pages=a.robots * blocks)
    else:
        memory = StreamMemory(c, a.robots, a.frames * n, max_frames=most)
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    with torch.no_grad():
        for f in range(a.frames):
            images, lang, state, noise = P.synthetic_observations(a.robots, c, seed=f)
            if a.candidates > 1:
                noise = torch.randn(a.robots * a.candidates, *noise.shape[1:], device=noise.device)
            ev[0].record()
            if window and memory.tokens == window * n:
                memory.keep_recent((window - 1) * n)
            actions = model(images, lang, state, noise, memory=memory)
            ev[1].record()
            ev[1].synchronize()
            print(f'frame {f}: {memory.tokens} tokens remembered, {ev[0].elapsed_time(ev[1]):.2f} ms, actions {tuple(actions.shape)}')
    print(f'memory: {memory.bytes / 2 ** 20:.1f} MiB for {a.robots} robots ({c.llm_layers} layers, 8 bits)')
    return actions


if __name__ == '__main__':
    main()
