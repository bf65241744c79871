"""A rolling forecast's time attention: patches arrive a few at a time, and each layer attends over what it has cached.

``RollingTimeAttention`` is one layer: the q|k|v projection (``ops.linear_device``), the new tokens' keys and values into
the layer's ``PagedCache`` with RoPE, their attention over the cache (sliding window and sinks), the output projection
and the residual. ``Pages`` hands the layers' pages to series as they grow and takes back those that a window has left
behind. Run as a command, it feeds series patch by patch and holds the result to the same layers fed all at once:

    python -m jitcast_b200.rolling [--bits 4] [--window 512 --sinks 4] [--series 64 --patches 700]
"""

from __future__ import annotations

import argparse

from . import ops
from .kvcache import PagedCache, Step, rope_table


class Pages:
    """Page numbers of a pool shared by the layers (page p of every layer's cache belongs together). ``grow`` and ``leave``
    work on the host and may run ahead of the GPU: a step enqueued after a ``grow`` reads the table of that ``grow``."""

    def __init__(self, series: int, pages: int, page_size: int, most_tokens: int, device="cuda"):
        import torch

        self.page_size, self.pages, self.free, self.peak = page_size, pages, list(range(pages - 1, -1, -1)), 0
        columns = -(-most_tokens // page_size)
        # [series, columns]: -1 where no page is, or no longer
        self.host = torch.full((series, columns), -1, dtype=torch.int32).numpy()
        self.table = torch.full((series, columns), -1, dtype=torch.int32, device=device)
        self.pinned = self.table.is_cuda
        self.given = [0] * series  # columns handed out so far; those that were left stay without a page
        self.left = [0] * series   # columns looked at for leaving

    @staticmethod
    def most(tokens: int, page_size: int, window: int = 0, sinks: int = 0, chunk: int = 1) -> int:
        """The most pages that a series of ``tokens`` holds when it grows by up to ``chunk`` at a time."""
        whole = -(-tokens // page_size)
        if not window:
            return whole
        # the sinks' pages, and a band of window - 1 + chunk tokens that starts anywhere in a page
        return min(whole, -(-sinks // page_size) + (window - 1 + chunk + page_size - 2) // page_size + 1)

    @property
    def used(self) -> int:
        return self.pages - len(self.free)

    def grow(self, lengths) -> None:
        """Pages for series of these lengths (host integers), taken from the free ones."""
        import torch

        need = [-(-length // self.page_size) for length in lengths]
        if sum(max(0, n - g) for n, g in zip(need, self.given)) > len(self.free):
            raise RuntimeError("the cache has no free page left")
        changed = False
        for s, n in enumerate(need):
            for c in range(self.given[s], n):
                self.host[s, c] = self.free.pop()
                changed = True
            self.given[s] = max(self.given[s], n)
        self.peak = max(self.peak, self.used)
        if changed:
            # a buffer of its own for each copy, which may run after the host's table has changed again
            now = torch.from_numpy(self.host).clone()
            self.table.copy_(now.pin_memory() if self.pinned else now, non_blocking=True)

    def leave(self, lengths, window: int, sinks: int) -> None:
        """Frees the pages that no later token of these series can see, for tokens of steps enqueued after this call."""
        if not window:
            return
        first = -(-sinks // self.page_size)
        for s, length in enumerate(lengths):
            last = min(max(0, length + 1 - window) // self.page_size, self.given[s])
            for c in range(max(first, self.left[s]), last):
                self.free.append(int(self.host[s, c]))
                self.host[s, c] = -1
            self.left[s] = max(self.left[s], last)


class RollingTimeAttention:
    """One layer: ``w_qkv`` [3d, d] (q|k|v, heads-major) and ``w_o`` [d, d], FP32 on the GPU."""

    def __init__(self, w_qkv, w_o, heads: int, pages: int, page_size: int = 64, bits: int = 16, window: int = 0,
                 sinks: int = 0, rope=None, pairs: int | None = None):
        import torch

        self.w_qkv, self.w_o, self.heads, self.window, self.sinks = w_qkv, w_o, heads, window, sinks
        self.dim = w_o.shape[0] // heads
        self.cache = PagedCache(pages, page_size, heads, self.dim, dtype=torch.float16 if bits == 16 else None, bits=bits,
                                device=w_o.device)
        self.rope, self.pairs = rope, pairs

    def __call__(self, x, step: Step):
        """x [tokens, d] FP32 of the step's new tokens -> x + attention(x)."""
        import torch

        n, d = x.shape
        qkv = torch.empty((n, 3 * d), dtype=torch.float32, device=x.device)
        ops.linear_device(x, self.w_qkv, None, qkv, 0, "fp16")
        # the FP16 of the engines: saturated
        q, k, v = qkv.clamp_(-65504.0, 65504.0).half().view(n, 3, self.heads, self.dim).unbind(1)
        q = self.cache.append(step, k, v, q=q, rope=self.rope, pairs=self.pairs)
        o = self.cache.attention(step, q, window=self.window, sinks=self.sinks)
        y = x.clone()
        ops.linear_device(o.view(n, d).float(), self.w_o, None, y, ops.ACCUMULATE, "fp16")
        return y


def run(layers, pages: Pages, tokens, chunks):
    """Feeds tokens [series, patches, d] through the layers, chunks[i] patches of every series at a time; returns the
    outputs [series, patches, d]."""
    import torch

    series, patches, d = tokens.shape
    start0 = torch.arange(series + 1, dtype=torch.int32, device=tokens.device)
    length = torch.zeros(series, dtype=torch.int32, device=tokens.device)
    out, done = [], 0
    for n in chunks:
        done += n
        length += n
        pages.grow([done] * series)
        step = Step(length, pages.table, done, None if n == 1 else start0 * n, n)
        x = tokens[:, done - n:done].reshape(series * n, d).contiguous()
        for layer in layers:
            x = layer(x, step)
        out.append(x.view(series, n, d))
        pages.leave([done] * series, layers[0].window, layers[0].sinks)
    return torch.cat(out, 1)


def demo(series=16, patches=300, prompt=130, heads=4, dim=64, depth=2, bits=16, window=0, sinks=0, page_size=64, seed=0):
    """(outputs fed patch by patch after a prompt, outputs of everything at once, most pages in use). The pool of the first
    holds what its window needs and no more."""
    import torch

    d, dev = heads * dim, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    weights = [(rand(3 * d, d) * d ** -0.5, rand(d, d) * d ** -0.5) for _ in range(depth)]
    tokens = rand(series, patches, d)
    rope = rope_table(patches, dim, dim // 4)

    def build(chunk):
        most = series * max(Pages.most(patches, page_size, window, sinks), Pages.most(chunk, page_size))
        return [RollingTimeAttention(wq, wo, heads, most, page_size, bits, window, sinks, rope, dim // 4)
                for wq, wo in weights], Pages(series, most, page_size, patches)

    layers, pages = build(prompt)
    rolled = run(layers, pages, tokens, [prompt] + [1] * (patches - prompt))
    used = pages.peak
    layers, pages = build(patches)
    return rolled, run(layers, pages, tokens, [patches]), used


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in dict(series=16, patches=300, prompt=130, heads=4, dim=64, depth=2, bits=16, window=0, sinks=0,
                            page_size=64, seed=0).items():
        p.add_argument(f"--{name.replace('_', '-')}", type=int, default=value)
    args = vars(p.parse_args())
    rolled, whole, used = demo(**args)
    ops.device_sync()
    err = float((rolled - whole).norm() / whole.norm())
    print(f"{args['series']} series of {args['patches']} patches, {args['prompt']} at once and then one by one: "
          f"{err:.2e} from all at once (relative, 2-norm); {used} pages in use at most")


if __name__ == "__main__":
    main()
