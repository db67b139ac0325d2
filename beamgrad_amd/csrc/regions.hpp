// SPDX-License-Identifier: MIT
//
// Whether the memory that one call writes in many workgroups at once lies apart:
// pools of a cache, states, and what is read meanwhile. Host code.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <numeric>
#include <utility>
#include <vector>

namespace dbs_hip {

// n[0] * n[1] rows of `bytes` bytes, at base + i * stride[0] + j * stride[1];
// no number is negative, and none is zero but the strides.
struct Region {
    uintptr_t base;
    int64_t n[2], stride[2], bytes;

    // Bytes that the rows of dimension d at one place of the other reach over; -1: more
    // than an address holds.
    int64_t run(int d) const {
        int64_t reach, all;
        return __builtin_mul_overflow(n[d] - 1, stride[d], &reach) || __builtin_add_overflow(reach, bytes, &all) ? -1 : all;
    }
    int64_t extent() const {
        int64_t reach, all;
        const int64_t inner = run(1);
        return inner < 0 || __builtin_mul_overflow(n[0] - 1, stride[0], &reach) || __builtin_add_overflow(reach, inner, &all) ||
                       static_cast<uint64_t>(all) > UINTPTR_MAX - base
                   ? -1
                   : all;
    }
    int64_t step(int d) const { return n[d] > 1 ? stride[d] : 0; }
    // Whether no two of its rows meet: one dimension's runs lie apart along the other.
    bool distinct() const {
        const auto nested = [&](int d) { return (n[d] == 1 || stride[d] >= run(1 - d)) && (n[1 - d] == 1 || stride[1 - d] >= bytes); };
        return extent() >= 0 && (nested(0) || nested(1));
    }
};

// Whether runs of `a` and `b` bytes that begin `off` apart, each again and again
// every `period` bytes, never meet.
inline bool apart_in_period(int64_t off, int64_t a, int64_t b, int64_t period) {
    return period > 0 && a >= 0 && b >= 0 && off >= a && b <= period && off <= period - b;
}

// Whether two regions have no byte in common. True is proven: their extents lie
// apart, or the runs along one dimension do within the other's common step, or
// the rows within all steps' (pools, or tokens, laid in turns in one buffer).
inline bool apart(const Region& a, const Region& b) {
    const int64_t length_a = a.extent(), length_b = b.extent();
    if (length_a < 0 || length_b < 0) return false;
    if (a.base + length_a <= b.base || b.base + length_b <= a.base) return true;
    const auto within = [&](int64_t period, int64_t run_a, int64_t run_b) {
        if (period <= 0) return false;
        const int64_t far = a.base <= b.base ? static_cast<int64_t>((b.base - a.base) % period)
                                             : (period - static_cast<int64_t>((a.base - b.base) % period)) % period;
        return apart_in_period(far, run_a, run_b, period);
    };
    const int64_t step0 = std::gcd(a.step(0), b.step(0)), step1 = std::gcd(a.step(1), b.step(1));
    return within(step0, a.run(1), b.run(1)) || within(step1, a.run(0), b.run(0)) || within(std::gcd(step0, step1), a.bytes, b.bytes);
}

// Two regions that may have a byte in common: `first` of the written ones, and
// `second` of the written ones (the same one: its own rows meet) or of those that
// are read. first < 0: there are none.
struct Meeting {
    int first = -1, second = -1;
    bool reads = false;
};

// Of the usual case alone, without memory of its own (a call's host work counts):
// written regions and read ones one after the other, by their addresses. False:
// find_meeting says. `written(i)` and `read(i)` make a region.
template <class Written, class Read>
bool in_order(int n, Written written, int m, Read read) {
    uintptr_t end = 0;
    for (int i = 0; i < n; ++i) {
        const Region r = written(i);
        if (!r.distinct() || r.base < end) return false;
        end = r.base + r.extent();
    }
    // the first written region that ends past the read one's begin
    int i = 0;
    uintptr_t last = 0;
    for (int j = 0; j < m; ++j) {
        const Region r = read(j);
        const int64_t length = r.extent();
        if (length < 0 || r.base < last) return false;
        last = r.base;
        for (; i < n; ++i) {
            const Region w = written(i);
            if (w.base + w.extent() <= r.base) continue;
            if (w.base < r.base + length) return false;
            break;
        }
    }
    return true;
}

// Many pools lie in one buffer in turns: that is settled without a comparison of
// every two.
inline Meeting find_meeting(const std::vector<Region>& written, const std::vector<Region>& read) {
    const int n = static_cast<int>(written.size());
    for (int i = 0; i < n; ++i)
        if (!written[i].distinct()) return {i, i, false};
    std::vector<int> order(n);
    std::iota(order.begin(), order.end(), 0);
    const auto before = [&](int i, int j) { return written[i].base < written[j].base; };
    if (!std::is_sorted(order.begin(), order.end(), before)) std::sort(order.begin(), order.end(), before);
    // members order[from, to) of a stretch of memory that their extents cover
    struct Stretch {
        uintptr_t base, end;
        int from, to;
    };
    std::vector<Stretch> stretches;
    stretches.reserve(n);
    for (int k = 0; k < n; ++k) {
        const Region& r = written[order[k]];
        const uintptr_t end = r.base + r.extent();
        if (!stretches.empty() && r.base < stretches.back().end) {
            stretches.back().end = std::max(stretches.back().end, end);
            stretches.back().to = k + 1;
        } else {
            stretches.push_back({r.base, end, k, k + 1});
        }
    }
    // members in turns, all with one step of dimension d (2: of both): their runs
    // in its order
    const auto in_turns = [&](const Stretch& s, int d) {
        const auto step = [&](const Region& r) { return d < 2 ? r.step(d) : std::gcd(r.step(0), r.step(1)); };
        const int64_t period = step(written[order[s.from]]);
        std::vector<std::pair<int64_t, int64_t>> runs;  // where it begins in the period, its length
        for (int k = s.from; k < s.to; ++k) {
            const Region& r = written[order[k]];
            if (period <= 0 || step(r) != period) return false;
            runs.emplace_back(static_cast<int64_t>((r.base - s.base) % period), d < 2 ? r.run(1 - d) : r.bytes);
        }
        std::sort(runs.begin(), runs.end());
        for (size_t k = 0; k < runs.size(); ++k) {
            const int64_t next = k + 1 < runs.size() ? runs[k + 1].first : runs[0].first + period;
            if (runs[k].second > next - runs[k].first) return false;
        }
        return true;
    };
    for (const Stretch& s : stretches) {
        if (s.to - s.from == 1 || in_turns(s, 0) || in_turns(s, 1) || in_turns(s, 2)) continue;
        for (int i = s.from; i < s.to; ++i)
            for (int j = i + 1; j < s.to; ++j)
                if (!apart(written[order[i]], written[order[j]]))
                    return {std::min(order[i], order[j]), std::max(order[i], order[j]), false};
    }
    for (int j = 0; j < static_cast<int>(read.size()); ++j) {
        const int64_t length = read[j].extent();
        if (length < 0) return {0, j, true};
        const uintptr_t end = read[j].base + length;
        auto s = std::upper_bound(stretches.begin(), stretches.end(), read[j].base, [](uintptr_t at, const Stretch& x) { return at < x.end; });
        for (; s != stretches.end() && s->base < end; ++s)
            for (int i = s->from; i < s->to; ++i)
                if (!apart(written[order[i]], read[j])) return {order[i], j, true};
    }
    return {};
}

template <class Written, class Read>
bool all_apart(int n, Written written, int m, Read read) {
    if (in_order(n, written, m, read)) return true;
    std::vector<Region> all_written, all_read;
    all_written.reserve(n);
    all_read.reserve(m);
    for (int i = 0; i < n; ++i) all_written.push_back(written(i));
    for (int j = 0; j < m; ++j) all_read.push_back(read(j));
    return find_meeting(all_written, all_read).first < 0;
}

}  // namespace dbs_hip
