"""numpy arrays laid out in one device arena, for tests of entry points that take offsets."""
import numpy as np


class Box:
    """put() reserves and remembers, place() writes everything, get() reads an array back."""

    def __init__(self, ql, ctx):
        self.lay, self.ctx, self.items, self.arena = ql.ArenaLayout(), ctx, {}, None

    def put(self, name, a, align=256, gap=0):
        """gap: bytes left before it, so that its offset is not a multiple of `align`."""
        a = np.ascontiguousarray(a)
        off = self.lay.take(a.nbytes + gap + 16, align) + gap
        self.items[name] = (off, a)
        return off

    def place(self):
        self.arena = self.ctx.arena(self.lay.used + 256)
        for off, a in self.items.values():
            if a.nbytes:
                self.arena.write(off, a)
        return self.arena

    def off(self, name):
        return self.items[name][0]

    def get(self, name):
        off, a = self.items[name]
        return self.arena.read(off, a.shape, a.dtype) if a.nbytes else a.copy()

    def release(self):
        self.arena.release()
