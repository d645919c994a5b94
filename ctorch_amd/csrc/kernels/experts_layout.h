// Where a row's entries lie as the experts' products read them (experts.hip).  Of the host and the device.
#pragma once

namespace dlk {

// Rows of a width that is no multiple of a piece's U entries (8 of bf16, 4 of f32): whole pieces, and then the row's last U
// entries, of which those that a piece holds already are zeros.  (The matrices' last piece is read so too.)
constexpr int laid_width(int width, int unit) { return (width + unit - 1) / unit * unit; }
constexpr int laid_place(int i, int width, int unit) {
    const int whole = width / unit * unit;
    return i < whole ? i : whole + i - (width - unit);
}

// A pair's hidden entries, in pieces (`laid`) or side by side: their room, the place of entry i, and the place that is zeroed with
// it, below zero if none.  Side by side there is no room for zeros: the next entry is another's.
constexpr int hidden_line(int hidden, int unit, bool laid) { return laid ? laid_width(hidden, unit) : hidden; }
constexpr int hidden_place(int i, int hidden, int unit, bool laid) { return laid ? laid_place(i, hidden, unit) : i; }
constexpr int hidden_zero(int i, int hidden, int unit, bool laid) {
    const int whole = hidden / unit * unit;
    return laid && hidden > whole && i >= hidden - unit && i < whole ? whole + i - (hidden - unit) : -1;
}

} // namespace dlk
