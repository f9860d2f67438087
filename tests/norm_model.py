"""The order of the sums of layer normalisation, in numpy's binary32 (one rounding per operation).

A row of N elements belongs to T = 4, 8, ... 1024 threads, the fewest that hold it in 16 elements each -- in a 16-bit type in 24, where
N is at most 3/4 (in the backward pass 9/16) of what those threads of 16 elements would hold, and that is more than 64.  A granule is 4 elements
(binary32) or 8 (16-bit types); granule i of thread j starts at element (i T + j) * granule, or as late as a whole granule
allows, and leaves out what an earlier one has.  A granule is summed in pairs and pairs of pairs, a thread's granules in turn,
the threads of a wave (64) as a butterfly, the waves in turn.  Sums over rows: runs of consecutive rows, one per workgroup; inside a
run the workgroup's teams take the rows in turn and their sums are added in the teams' order; then 16 sums of every 16th run are
added in order.  At most 256 rows: one sixteenth of the workgroup's threads as many sums, each of every so-many-th row in turn, added
in order.  (Rows of at most 16384 elements.)"""
import numpy as np

f32 = np.float32


def _pairs(v):
    """sum over the last axis, neighbours first"""
    while v.shape[-1] > 1:
        v = (v[..., 0::2] + v[..., 1::2]).astype(f32)
    return v[..., 0]


def _in_turn(v, axis):
    v = np.moveaxis(v, axis, 0)
    s = v[0]
    for t in v[1:]:
        s = (s + t).astype(f32)
    return s


class _Rows:
    """threads and granules of a row of n elements"""

    def __init__(self, n, granule, backward):
        self.threads = 4
        while self.threads * 16 < n:
            self.threads *= 2
        each, padded = 16, self.threads * 16
        if granule == 8 and padded > 64 and (16 * n <= 9 * padded if backward else 4 * n <= 3 * padded):
            each, self.threads = 24, 4
            while self.threads * 24 < n:
                self.threads *= 2
        g, t = granule, self.threads
        tiny = n < g
        c = (np.arange(each // g)[:, None] * t + np.arange(t)[None, :]) * g
        start = np.zeros_like(c) if tiny else np.minimum(c, n - g)
        at = start[..., None] + np.arange(g)
        self.used = (np.arange(g) >= np.minimum(c - start, g)[..., None]) & (at < n)
        self.at = np.minimum(at, n - 1)

    def sum(self, v):
        v = np.where(self.used, v[:, self.at], f32(0)).astype(f32)      # [rows, granules, threads, granule]
        v = _pairs(v)
        s = np.zeros(v.shape[:1] + v.shape[2:], f32)
        for i in range(v.shape[1]):
            s = (s + v[:, i]).astype(f32)
        wave = min(64, self.threads)
        return _in_turn(_pairs(s.reshape(len(s), -1, wave)), 1)


class LayerNorm:
    def __init__(self, rows, cols, granule):
        self.rows, self.cols = rows, cols
        self.ahead, self.back = _Rows(cols, granule, False), _Rows(cols, granule, True)
        self.scale = f32(1.0 / cols)

    def forward(self, x, w, b, eps):
        mean = (self.ahead.sum(x) * self.scale).astype(f32)
        d = (x - mean[:, None]).astype(f32)
        var = (self.ahead.sum((d * d).astype(f32)) * self.scale).astype(f32)
        rstd = (f32(1) / np.sqrt((var + f32(eps)).astype(f32)).astype(f32)).astype(f32)
        xh = (d * rstd[:, None]).astype(f32)
        return ((xh * w).astype(f32) + b).astype(f32), mean, rstd, xh

    def over_rows(self, v):
        threads = max(256, self.back.threads)
        if self.rows <= 256:
            groups = threads // 16
            parts = np.zeros((groups, self.cols), f32)
            for r in range(self.rows):
                parts[r % groups] = (parts[r % groups] + v[r]).astype(f32)
            return _in_turn(parts, 0)
        teams = threads // self.back.threads
        run = max(4, -(-self.rows // (512 if self.back.threads < 512 and self.rows >= 4096 else 256)))
        run = -(-run // teams) * teams
        runs = []
        for r0 in range(0, self.rows, run):
            part = v[r0:r0 + run]
            sums = np.zeros((teams, self.cols), f32)
            for r in range(len(part)):
                sums[r % teams] = (sums[r % teams] + part[r]).astype(f32)
            runs.append(_in_turn(sums, 0))
        parts = np.zeros((16, self.cols), f32)
        for i, s in enumerate(runs):
            parts[i % 16] = (parts[i % 16] + s).astype(f32)
        return _in_turn(parts, 0)

    def backward(self, gy, xh, rstd, w):
        g = (gy * w).astype(f32)
        c1 = (self.back.sum(g) * self.scale).astype(f32)[:, None]
        c2 = (self.back.sum((g * xh).astype(f32)) * self.scale).astype(f32)[:, None]
        gx = (rstd[:, None] * ((g - c1).astype(f32) - (xh * c2).astype(f32)).astype(f32)).astype(f32)
        return gx, self.over_rows((gy * xh).astype(f32)), self.over_rows(gy)
