// Host side of the grammar operators: the bytes of a vocabulary's tokens.
#pragma once
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../../include/zbpe.h"

namespace zbpe {

// The tokens' lengths and an order in which every token comes after its halves (decode's rules: a token below 256 is its
// byte, any other the first merge that makes it). Iterative: a table read from a file may nest as deep as it is long.
struct VocabTree {
    struct Node {
        int32_t a = -1, b = -1;  // halves; -1: no merge makes this id
    };
    std::vector<Node> node;
    std::vector<uint64_t> len;
    std::vector<uint32_t> order;  // ids from 256 on that have bytes, halves first
    uint64_t total = 0;
    std::string err;

    zbpe_status build(const uint16_t *triples, size_t n_merges, size_t vocab_size) {
        node.assign(vocab_size, Node{});
        len.assign(vocab_size, 0);
        for (size_t v = 0; v < 256; v++) len[v] = 1;
        for (size_t i = 0; i < n_merges; i++) {
            const uint16_t *t = triples + 3 * i;
            if (t[2] >= vocab_size) {
                err = "merge " + std::to_string(i) + " makes token " + std::to_string(t[2]) + ", outside a vocabulary of " + std::to_string(vocab_size);
                return ZBPE_INVALID_ARGUMENT;
            }
            if (t[2] < 256 || node[t[2]].a >= 0) continue;
            node[t[2]] = Node{t[0], t[1]};
        }
        constexpr uint64_t MOST = (1ull << 31) - 1;
        std::vector<uint8_t> open(vocab_size, 0);  // 1: on the path from the root, 2: done
        std::vector<uint32_t> path;
        for (size_t v = 256; v < vocab_size; v++) {
            if (node[v].a < 0 || open[v] == 2) continue;
            path.push_back((uint32_t)v);
            while (!path.empty()) {
                const uint32_t x = path.back();
                open[x] = 1;
                uint32_t child = 0;
                for (int32_t h : {node[x].a, node[x].b}) {
                    if (h < 256) continue;
                    const bool made = (size_t)h < vocab_size && node[h].a >= 0;
                    if (!made || open[h] == 1) {
                        err = "token " + std::to_string(x) + " is made from token " + std::to_string(h) +
                              (made ? ", which is made from it" : ", which no merge makes");
                        return ZBPE_INVALID_TOKEN;
                    }
                    if (open[h] == 2) continue;
                    child = (uint32_t)h;
                    break;
                }
                if (child) {
                    path.push_back(child);
                    continue;
                }
                len[x] = len[node[x].a] + len[node[x].b];
                if (len[x] > MOST) {
                    err = "token " + std::to_string(x) + " has 2^31 bytes or more";
                    return ZBPE_INVALID_ARGUMENT;
                }
                open[x] = 2;
                order.push_back(x);
                path.pop_back();
            }
        }
        for (uint64_t l : len) total += l;
        if (total > MOST) {
            err = "the tokens have 2^31 bytes or more";
            return ZBPE_INVALID_ARGUMENT;
        }
        return ZBPE_OK;
    }

    void write(uint32_t *offsets, uint8_t *bytes) const {
        uint64_t at = 0;
        for (size_t v = 0; v < len.size(); v++) {
            offsets[v] = (uint32_t)at;
            at += len[v];
        }
        offsets[len.size()] = (uint32_t)at;
        if (!bytes) return;
        for (size_t v = 0; v < 256; v++) bytes[offsets[v]] = (uint8_t)v;
        for (uint32_t v : order) {
            uint8_t *to = bytes + offsets[v];
            const uint32_t a = (uint32_t)node[v].a, b = (uint32_t)node[v].b;
            for (uint64_t i = 0; i < len[a]; i++) to[i] = bytes[offsets[a] + i];
            for (uint64_t i = 0; i < len[b]; i++) to[len[a] + i] = bytes[offsets[b] + i];
        }
    }
};

// The index that grammar masks read: the tokens of each INDEX_SLICE neighbouring ids in the order of their bytes, those without
// bytes last, padded to whole waves. Heads, then tails (a token's bytes, as far as they fit), then for each 64 tokens the least
// and the largest first byte.
constexpr int INDEX_SLICE = 8192, INDEX_HEAD = 5, INDEX_BYTES = INDEX_HEAD + 16;

#ifdef __HIP__
#define ZBPE_BOTH __host__ __device__
#else
#define ZBPE_BOTH
#endif

// Bytes that grammars seldom tell apart share a class; punctuation, spaces and line ends have classes of their own. (Any
// classes give the same masks: these decide how often a token's set shows that it leaves a state as it is.)
ZBPE_BOTH constexpr int byte_class(int b) {
    return b >= 0x80                ? (b >= 0xc0 ? 1 : 0)
           : b >= '0' && b <= '9'   ? 2
           : b >= 'A' && b <= 'F'   ? 3
           : b >= 'G' && b <= 'Z'   ? 4
           : b >= 'a' && b <= 'f'   ? 5
           : b >= 'g' && b <= 'z'   ? 6
           : b == '\t'              ? 7
           : b == '\n'              ? 8
           : b == '\r'              ? 9
           : b < 32 || b == 127     ? 10
           : b < '0'                ? 11 + b - 32   // 11 .. 26
           : b < 'A'                ? 27 + b - ':'  // 27 .. 33
           : b < 'a'                ? 34 + b - '['  // 34 .. 39
                                    : 40 + b - '{'; // 40 .. 43
}

struct IndexHead {
    uint32_t classes[2];  // one bit for each class among its bytes
    uint32_t what;        // id from the slice's first; length << 16 (0: padding; INDEX_BYTES + 1: longer); the first byte << 24
    uint32_t more;        // four bytes more
    ZBPE_BOTH int id() const { return (int)(what & 0xffff); }
    ZBPE_BOTH int length() const { return (int)(what >> 16 & 0xff); }
    ZBPE_BOTH int byte(int j) const { return (int)(j ? more >> (8 * (j - 1)) & 0xff : what >> 24); }
};
struct IndexTail {
    uint32_t word[4];
    ZBPE_BOTH int byte(int j) const { return (int)(word[j >> 2] >> (8 * (j & 3)) & 0xff); }
};
struct IndexBounds {
    uint8_t lo, hi;  // lo > hi: none of the 64 has bytes
};
struct IndexView {
    const IndexHead *heads;
    const IndexTail *tails;
    const IndexBounds *bounds;
    ZBPE_BOTH IndexView(const void *index, int vocab) {
        const size_t n = ((size_t)vocab + 63) / 64 * 64;
        heads = (const IndexHead *)index;
        tails = (const IndexTail *)(heads + n);
        bounds = (const IndexBounds *)(tails + n);
    }
};
constexpr size_t index_size(size_t vocab) { return (vocab + 63) / 64 * (64 * (sizeof(IndexHead) + sizeof(IndexTail)) + sizeof(IndexBounds)); }

inline void index_tokens(const uint32_t *offsets, const uint8_t *bytes, size_t vocab_size, void *index) {
    const IndexView view(index, (int)vocab_size);
    IndexHead *heads = const_cast<IndexHead *>(view.heads);
    IndexTail *tails = const_cast<IndexTail *>(view.tails);
    IndexBounds *bounds = const_cast<IndexBounds *>(view.bounds);
    memset(index, 0, index_size(vocab_size));
    std::vector<std::pair<uint64_t, uint32_t>> ids;  // a token's first eight bytes, larger for a later place, and its id
    for (size_t base = 0; base < vocab_size; base += INDEX_SLICE) {
        const size_t end = std::min(vocab_size, base + INDEX_SLICE);
        ids.clear();
        for (size_t v = base; v < end; v++) {
            uint64_t key = 0;
            for (uint32_t i = offsets[v]; i < offsets[v + 1] && i < offsets[v] + 8; i++) key |= (uint64_t)bytes[i] << (56 - 8 * (i - offsets[v]));
            if (offsets[v] < offsets[v + 1]) ids.push_back({key, (uint32_t)v});
        }
        std::sort(ids.begin(), ids.end());
        for (size_t i = 0; i < ids.size(); i++) {
            const uint32_t v = ids[i].second, at = offsets[v], n = offsets[v + 1] - at;
            uint64_t classes = 0;
            for (uint32_t j = 0; j < n; j++) classes |= 1ull << byte_class(bytes[at + j]);
            uint8_t data[INDEX_BYTES] = {};
            memcpy(data, bytes + at, std::min<uint32_t>(n, INDEX_BYTES));
            IndexHead &h = heads[base + i];
            h.classes[0] = (uint32_t)classes;
            h.classes[1] = (uint32_t)(classes >> 32);
            h.what = (uint32_t)(v - base) | std::min<uint32_t>(n, INDEX_BYTES + 1) << 16 | (uint32_t)data[0] << 24;
            memcpy(&h.more, data + 1, 4);
            memcpy(tails[base + i].word, data + INDEX_HEAD, 16);
        }
        for (size_t i = 0; i < end - base; i += 64) {
            const size_t last = std::min(i + 63, ids.size() - 1);
            bounds[(base + i) / 64] = i < ids.size() ? IndexBounds{bytes[offsets[ids[i].second]], bytes[offsets[ids[last].second]]} : IndexBounds{255, 0};
        }
    }
}

}  // namespace zbpe
