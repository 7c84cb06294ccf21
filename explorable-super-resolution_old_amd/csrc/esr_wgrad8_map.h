// Which part of the 8-bit weight gradient (esr_wgrad8.hip) a workgroup takes: a split of the pixels and one of its `work`
// items (64 ci × 64 co × a tap group).  Workgroup ids go round the 8 XCDs.  Eight splits at a time, each split's items,
// which read the same pixels, go to one XCD and its L2; the last splits % 8 are spread over all of them, item by item
// (tied to an XCD each they left the others idle: 512 -> 100 channels, 8×8, 4 splits, 342 us on four XCDs).
#pragma once

namespace wgrad8 {

struct Place {
    int split, item;
};

constexpr Place place(int id, int splits, int work) {
    const int whole = splits / 8 * 8 * work, r = id - whole;
    return r < 0 ? Place{id / 8 / work * 8 + id % 8, id / 8 % work} : Place{splits / 8 * 8 + r / work, r % work};
}

}  // namespace wgrad8
