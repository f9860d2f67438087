"""Layer normalisation's offset rows in numpy's binary32, in the order of norm_model: rows whose mean is more than 16 times their spread are
centred in two numbers, the mean (once more corrected by the mean of what it leaves) and the mean of what the corrected one leaves."""
import numpy as np

import norm_model

f32 = np.float32


class LayerNorm(norm_model.LayerNorm):
    def __init__(self, rows, cols, granule):
        super().__init__(rows, cols, granule)
        self.granule = granule

    def _mean(self, rows, v):
        return (rows.sum(v) * self.scale).astype(f32)

    def forward(self, x, w, b, eps):
        mean = self._mean(self.ahead, x)
        d = (x - mean[:, None]).astype(f32)
        var = self._mean(self.ahead, (d * d).astype(f32))
        offset = (mean * mean).astype(f32) > (f32(256) * var).astype(f32)
        better = np.where(offset, (mean + self._mean(self.ahead, d)).astype(f32), mean)
        d = (d - (better - mean).astype(f32)[:, None]).astype(f32)
        mean = better
        rest = np.where(offset, self._mean(self.ahead, d), f32(0))
        d = (d - rest[:, None]).astype(f32)
        var = self._mean(self.ahead, (d * d).astype(f32))
        rstd = (f32(1) / np.sqrt((var + f32(eps)).astype(f32)).astype(f32)).astype(f32)
        xh = (d * rstd[:, None]).astype(f32)
        return ((xh * w).astype(f32) + b).astype(f32), mean, rstd, offset

    def backward(self, gy, x, mean, rstd, w):
        offset = (np.abs(mean) * rstd).astype(f32) > f32(16)
        d = (x - mean[:, None]).astype(f32)

        def xh(total):
            rest = np.where(offset, (total * self.scale).astype(f32), f32(0))
            return ((d - rest[:, None]).astype(f32) * rstd[:, None]).astype(f32)

        rows = xh(self.back.sum(d))
        gx, gw, gb = super().backward(gy, rows, rstd, w)
        if self.rows <= 256:  # the sums over few rows make their own: a wave a row
            gw = self.over_rows((gy * xh(self._wave_sum(d))).astype(f32))
        return gx, gw, gb

    def _wave_sum(self, v):
        g = self.granule
        v = np.pad(v, ((0, 0), (0, -v.shape[1] % (64 * g)))).reshape(len(v), -1, 64, g)
        s = norm_model._in_turn(norm_model._pairs(v), 1)
        return norm_model._pairs((f32(0) + s).astype(f32))
