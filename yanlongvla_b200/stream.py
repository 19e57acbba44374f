"""A policy that acts on a stream of frames: every LLM layer keeps the keys and values of past frames in an 8-bit paged cache
(kernels.KV8Cache), positions have three axes (time, row, column), and a new frame's tokens attend to all that is remembered.

    python -m yanlongvla_b200.stream --robots 2 --frames 8 [--llm-layers 24]

runs the policy of `policy` (random weights, synthetic frames) with a memory and prints the time per frame. The kernels:
rope_axes turns the queries, kv8_append turns and stores the keys and stores the values, kv8_attention reads the cache. All
lengths and positions live on the device, so a step can be captured in a CUDA graph: what a capture records moves them on at each
replay, and StreamMemory.reserve(), called before each replay, keeps the host's count and checks the capacity.
"""
import argparse

import torch

from . import kernels as K


class StreamMemory:
    """Caches of every LLM layer for `robots` sequences of up to `max_tokens` tokens. Pages are assigned once: block i of robot b
    is page b * blocks + i of each layer. Its operators are the kernels in every runtime of the policy, the one of PyTorch
    operations among them."""

    def __init__(self, c, robots, max_tokens, device='cuda', theta=10000.0, max_frames=4096):
        D = c.llm_hidden // c.llm_heads
        self.c, self.robots, self.max_tokens, self.tokens = c, robots, max_tokens, 0
        blocks = -(-max_tokens // K.KV8_BLOCK)
        self.caches = [K.KV8Cache.empty(robots * blocks, c.llm_kv_heads, D, device) for _ in range(c.llm_layers)]
        self.table = torch.arange(robots * blocks, dtype=torch.int32, device=device).view(robots, blocks)
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

    def reserve(self):
        """Count the next frame in on the host; refused where it does not fit. begin_frame calls it, except in a capture, which runs
        nothing: call it before each replay of a captured step."""
        n = self.pos.shape[2]
        if self.tokens + n > self.max_tokens or self.frames >= self.max_frames:
            raise K.TcqError(f'StreamMemory: a frame of {n} tokens does not fit behind {self.tokens} of {self.max_tokens} tokens, {self.frames} frames')
        self.frames += 1
        self.tokens += n

    def begin_frame(self, frame=None):
        """Make room for the next frame: its tokens follow those remembered. On the device but for the check of the capacity.
        frame: the (B, T, ...) tensor that the layers will get; one of another batch or length is refused before anything moves."""
        n = self.pos.shape[2]
        if frame is not None and tuple(frame.shape[:2]) != (self.robots, n):
            raise K.TcqError(f'StreamMemory: a frame of {self.robots} robots with {n} tokens each expected, got {tuple(frame.shape[:2])}')
        if not torch.cuda.is_current_stream_capturing():
            self.reserve()
        self.pos[0] += 1
        self.start.copy_(self.lens)
        self.lens += n

    def attend(self, layer, q, k, v):
        """The attention of one layer over everything remembered and the current frame (causal): q (B, T, heads * D) is turned in
        place, k and v (B, T, kv_heads * D) go into the layer's cache."""
        cache = self.caches[layer]
        K.kv8_append(cache, k, v, self.table, self.start, rope=self.rope, pos=self.pos)
        K.rope_axes(q, self.pos, self.rope, out=q)
        return K.kv8_attention(q, cache, self.table, self.lens)

    def forget(self):
        self.tokens = self.frames = 0
        self.lens.zero_()
        self.start.zero_()
        self.pos[0].fill_(-1)

    @property
    def bytes(self):
        return sum(t.numel() * t.element_size() for c in self.caches for t in (c.k, c.v, c.k_scale, c.v_scale))


def main(argv=None):
    from . import policy as P
    ap = argparse.ArgumentParser(description='run the policy on a stream of synthetic frames with an 8-bit memory')
    ap.add_argument('--robots', type=int, default=1)
    ap.add_argument('--frames', type=int, default=16)
    ap.add_argument('--vit-layers', type=int, default=P.PolicyConfig.vit_layers)
    ap.add_argument('--llm-layers', type=int, default=P.PolicyConfig.llm_layers)
    ap.add_argument('--dit-layers', type=int, default=P.PolicyConfig.dit_layers)
    a = ap.parse_args(argv)
    c = P.PolicyConfig(vit_layers=a.vit_layers, llm_layers=a.llm_layers, dit_layers=a.dit_layers)
    model, _, _ = P.build_policy(runtime='resident', c=c)
    memory = StreamMemory(c, a.robots, a.frames * c.prefix_tokens)
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    with torch.no_grad():
        for f in range(a.frames):
            obs = P.synthetic_observations(a.robots, c, seed=f)
            ev[0].record()
            actions = model(*obs, memory=memory)
            ev[1].record()
            ev[1].synchronize()
            print(f'frame {f}: {memory.tokens} tokens remembered, {ev[0].elapsed_time(ev[1]):.2f} ms, actions {tuple(actions.shape)}')
    print(f'memory: {memory.bytes / 2 ** 20:.1f} MiB for {a.robots} robots ({c.llm_layers} layers, 8 bits)')
    return actions


if __name__ == '__main__':
    main()
